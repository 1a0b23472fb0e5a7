"""Serving operators over the C ABI: a paged key/value cache in 8 bits, the attention that
reads it, and sampling.

* :func:`reserve_slots` / :func:`release_slots` — block tables and slot maps, built on the
  GPU from the rows' lengths
* :func:`append_cache`    — keys and values of new tokens into their slots, e4m3 with one
  power-of-two scale per page and kv head
* :func:`cache_attention` — window-and-landmark (or full) attention of one or a few query
  tokens per sequence over the cache
* :func:`sample_tokens`   — temperature, top-k, top-p and min-p from given uniforms

:class:`PagedCache` holds the state of several sequences for a decoder stack and makes these
calls for it (:meth:`dsalt_b200.model.DSALTLMHeadModel.generate`).

The reference has no counterpart (it recomputes the whole sequence for every token). As in
:mod:`dsalt_b200.ops`, tensors must be CUDA tensors and every call launches on the current
stream of their device; lengths and tables stay on the device, so the operators do not
synchronise and every call can be captured into a CUDA graph. They are for answering, not for
training: no gradient goes through them.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _lib as L
from . import ops
from .ops import _dt, _ptr, _workspace

PAGE_SIZES = (16, 32, 64, 128)
HEAD_SIZES = (64, 128)
MAX_ROWS = 8192          # rows (sequences) of one call
MAX_VOCAB = 1 << 20
MAX_POSITIONS = 0x7fffff00  # of a row, and of the pool times its kv heads


class SlotPlan(NamedTuple):
    """What :func:`reserve_slots` found for the new tokens, packed row after row."""
    slots: torch.Tensor      # [n_tokens] int64: page * page_size + offset, -1 = none
    positions: torch.Tensor  # [n_tokens] int32: position within the sequence (0 where no slot)
    cu_new: torch.Tensor     # [S + 1] int32: first token of each row
    granted: torch.Tensor    # [S] bool
    seq_lens: torch.Tensor   # [S] int32: lengths with the new tokens of granted rows
    n_free: torch.Tensor     # [1] int32: pages left


def _on_one_device(first: torch.Tensor, *rest) -> torch.device:
    index = first.get_device()
    if index < 0:
        raise RuntimeError("dsalt_b200 operators need CUDA tensors (no CPU path)")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"tensors on {first.device} and {t.device} in one call")
    return first.device


def _want(t: torch.Tensor, name: str, dtype: torch.dtype, shape) -> None:
    if t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _run(dev: torch.device, name: str, *args) -> None:
    """The C call on the current stream of the tensors' device."""
    index = dev.index
    if index == torch._C._cuda_getDevice():
        L.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            L.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


@functools.lru_cache(maxsize=1024)
def _attention_workspace(T: int, S: int, H: int, n_kv: int, D: int) -> int:
    return L.query("dsalt_cache_attention_workspace_bytes", T, S, H, n_kv, D)


# --------------------------------------------------------------------------- slots
def reserve_slots(block_tables, seq_lens, new_lens, free_pages, n_free, page_size: int, n_tokens: int, *,
                  inplace: bool = False) -> SlotPlan:
    """Pages and slots for ``new_lens [S]`` more tokens of rows that hold ``seq_lens [S]``.

    ``block_tables [S, max_pages]`` int32 is extended in place with pages from the top of the
    stack ``free_pages [N]`` (the first ``n_free [1]`` entries count). Rows are served in
    order; a row whose table, or the room for ``n_tokens`` tokens, or the pool does not hold
    its new tokens is not granted: it keeps its length and its tokens get slot -1. A row that
    needs no page is not held up by rows that wait for one. With ``inplace`` the new lengths
    and free count are written to ``seq_lens`` and ``n_free`` (as a captured step needs)."""
    dev = _on_one_device(block_tables, seq_lens, new_lens, free_pages, n_free)
    if block_tables.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_tables must be [S, max_pages] and free_pages [N]")
    S, max_pages = block_tables.shape
    i32 = torch.int32
    _want(block_tables, "block_tables", i32, (S, max_pages))
    _want(seq_lens, "seq_lens", i32, (S,))
    _want(new_lens, "new_lens", i32, (S,))
    _want(free_pages, "free_pages", i32, free_pages.shape)
    _want(n_free, "n_free", i32, (1,))
    n_tokens = int(n_tokens)
    if n_tokens < 0:
        raise ValueError("n_tokens must not be negative")
    slots = torch.empty(n_tokens, dtype=torch.int64, device=dev)
    granted = torch.empty(S, dtype=torch.bool, device=dev)
    if inplace:
        positions, cu_new = torch.empty(n_tokens + S + 1, dtype=i32, device=dev).split_with_sizes((n_tokens, S + 1))
        lens, left = seq_lens, n_free
    else:
        positions, cu_new, lens, left = torch.empty(n_tokens + 2 * S + 2, dtype=i32, device=dev).split_with_sizes(
            (n_tokens, S + 1, S, 1))
    _run(dev, "dsalt_reserve_slots", block_tables.data_ptr(), S, max_pages, seq_lens.data_ptr(), new_lens.data_ptr(),
         free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), int(page_size), n_tokens, slots.data_ptr(),
         positions.data_ptr(), cu_new.data_ptr(), granted.data_ptr(), lens.data_ptr(), left.data_ptr())
    return SlotPlan(slots, positions, cu_new, granted, lens, left)


def release_slots(block_tables, seq_lens, release, free_pages, n_free, page_size: int) -> None:
    """Gives the pages of the rows flagged in ``release [S]`` bool back to the stack, in place:
    their table entries become -1 and their lengths 0. Pages go back in the order in which
    :func:`reserve_slots` would take them again. Rows that share a page are not counted: each
    flagged row gives back every page of its table."""
    dev = _on_one_device(block_tables, seq_lens, release, free_pages, n_free)
    if block_tables.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("block_tables must be [S, max_pages] and free_pages [N]")
    S, max_pages = block_tables.shape
    i32 = torch.int32
    _want(block_tables, "block_tables", i32, (S, max_pages))
    _want(seq_lens, "seq_lens", i32, (S,))
    _want(release, "release", torch.bool, (S,))
    _want(free_pages, "free_pages", i32, free_pages.shape)
    _want(n_free, "n_free", i32, (1,))
    _run(dev, "dsalt_release_slots", block_tables.data_ptr(), S, max_pages, seq_lens.data_ptr(), release.data_ptr(),
         free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), int(page_size))


# --------------------------------------------------------------------------- cache
def _cache_shapes(k_cache, v_cache, k_scale, v_scale):
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be [n_pages, H_kv, page_size, head_dim]")
    n_pages, n_kv, page, D = k_cache.shape
    _want(k_cache, "k_cache", torch.float8_e4m3fn, k_cache.shape)
    _want(v_cache, "v_cache", torch.float8_e4m3fn, k_cache.shape)
    _want(k_scale, "k_scale", torch.float32, (n_pages, n_kv))
    _want(v_scale, "v_scale", torch.float32, (n_pages, n_kv))
    return n_pages, n_kv, page, D


def _rows(x, packed: bool = False):
    """``x [T, H, D]``, its token and head strides, as 16-byte loads can take its rows (``packed``: a
    token's heads must follow one another, and its row must not overlap the next); else a copy."""
    T, H, D = x.shape
    if x.data_ptr() % 16 == 0:
        if x.is_contiguous():  # strides of single tokens or heads may be anything
            return x, H * D, D
        es, (token, head, one) = x.element_size(), x.stride()
        if T == 1:
            token = H * D
        if H == 1:
            head = D
        if one == 1 and token * es % 16 == 0 and head * es % 16 == 0 and not (packed and (head != D or token < H * D)):
            return x, token, head
    return x.clone(memory_format=torch.contiguous_format), H * D, D


def append_cache(k, v, k_cache, v_cache, k_scale, v_scale, slots) -> None:
    """Quantises ``k, v [T, H_kv, D]`` into their slots, in place.

    ``k_cache, v_cache [n_pages, H_kv, page_size, D]`` float8_e4m3fn, ``k_scale, v_scale
    [n_pages, H_kv]`` fp32 powers of two; ``slots [T]`` int64 from :func:`reserve_slots` (-1: the
    token is left out). The slots of one page must be distinct and lie within ``page_size``
    consecutive tokens of the call (:func:`reserve_slots` numbers them next to each other).
    The scale of a page follows the largest magnitude written since its first token; when it
    grows, the bytes already there are rescaled."""
    dev = _on_one_device(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    n_pages, n_kv, page, D = _cache_shapes(k_cache, v_cache, k_scale, v_scale)
    T = k.shape[0]
    if tuple(k.shape) != (T, n_kv, D) or v.shape != k.shape:
        raise ValueError(f"k and v must be [T, {n_kv}, {D}]")
    if v.dtype != k.dtype:
        raise TypeError("k and v must share a dtype")
    _want(slots, "slots", torch.int64, (T,))
    k, k_token, k_head = _rows(k)
    v, v_token, v_head = _rows(v)
    _run(dev, "dsalt_append_cache", k.data_ptr(), v.data_ptr(), _dt(k), T, n_kv, D, k_token, k_head, v_token, v_head,
         k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n_pages, page, slots.data_ptr())


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, *, cu_q=None, w_sizes=None,
                    lmk_indices=None, lmk_bias=None, out_dtype=None, return_lse: bool = False):
    """Attention of the last query tokens of each sequence over the cache: ``out [T, H, D]`` in
    ``out_dtype`` (default the query's), with ``return_lse`` also ``lse [T, H]`` fp32.

    ``seq_lens [S]`` int32 tokens in the cache, the query tokens included. ``cu_q [S + 1]`` int32
    (from 0, not falling) packs the query tokens, rows behind its last entry come out as zeros;
    without it there is one per sequence. With ``w_sizes [T]`` int32 the
    query at position ``i`` attends to its window ``[i - w + 1, i]`` and to the landmarks
    ``lmk_indices [H, S, k]`` before it, as :func:`dsalt_b200.ops.dsalt_attention` does
    (``lmk_bias`` is added to their logits); without, to ``[0, i]``. The scales may be any
    positive numbers, or 0, not only the powers of two that :func:`append_cache` writes."""
    dev = _on_one_device(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, w_sizes, lmk_indices,
                         lmk_bias)
    n_pages, n_kv, page, D = _cache_shapes(k_cache, v_cache, k_scale, v_scale)
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] % n_kv:
        raise ValueError(f"q must be [T, H, {D}] with H a multiple of {n_kv}")
    T, H, _ = q.shape
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [S, max_pages]")
    S, max_pages = block_tables.shape
    i32 = torch.int32
    _want(block_tables, "block_tables", i32, (S, max_pages))
    _want(seq_lens, "seq_lens", i32, (S,))
    if cu_q is not None:
        _want(cu_q, "cu_q", i32, (S + 1,))
    elif T != S:
        raise ValueError(f"{T} query tokens for {S} sequences: pass cu_q")
    if w_sizes is not None:
        _want(w_sizes, "w_sizes", i32, (T,))
    k_lmk = 0
    if lmk_indices is not None:
        if w_sizes is None:
            raise ValueError("landmarks need w_sizes")
        k_lmk = lmk_indices.shape[-1]
        _want(lmk_indices, "lmk_indices", i32, (H, S, k_lmk))
    if lmk_bias is not None:
        if lmk_indices is None:
            raise ValueError("lmk_bias needs lmk_indices")
        _want(lmk_bias, "lmk_bias", torch.float32, (H, S, k_lmk))
    q, q_stride, _ = _rows(q, packed=True)
    if (out_dtype is None or out_dtype is q.dtype) and q_stride == H * D:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        out = torch.empty(T, H, D, dtype=out_dtype or q.dtype, device=dev)
    lse = torch.empty(T, H, dtype=torch.float32, device=dev) if return_lse else None
    ws = _workspace(_attention_workspace(T, S, H, n_kv, D), dev)
    _run(dev, "dsalt_cache_attention", q.data_ptr(), _dt(q), T, H, n_kv, D, q_stride, k_cache.data_ptr(),
         v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n_pages, page, block_tables.data_ptr(), max_pages,
         seq_lens.data_ptr(), S, _ptr(cu_q), _ptr(w_sizes), _ptr(lmk_indices), _ptr(lmk_bias), k_lmk, out.data_ptr(),
         _dt(out), _ptr(lse), ws.data_ptr(), ws.numel())
    return (out, lse) if return_lse else out


# --------------------------------------------------------------------------- sampling
def _setting(v, name: str, B: int, dtype: torch.dtype, lo, hi):
    """(device array or None, number) of a setting given per row or for all."""
    if isinstance(v, torch.Tensor):
        _want(v, name, dtype, (B,))
        return v, 0
    if not lo <= v <= hi:  # refuses NaN as well
        raise ValueError(f"{name} must lie in [{lo}, {hi}], got {v}")
    return None, v


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprob: bool = False):
    """One token per row of ``logits [B, V]`` from the given uniforms ``u [B]`` fp32 in [0, 1):
    ``token [B]`` int64, with ``return_logprob`` also its log-probability ``[B]`` fp32 in the
    distribution that it was drawn from.

    Of the weights ``exp((l - max l) / temperature)`` ``top_k`` keeps the largest (equal logits:
    lowest index first; 0 = off), ``top_p`` of those the shortest prefix whose mass reaches
    ``top_p`` of theirs, ``min_p`` of those the weights of at least ``min_p``; the first of the
    order always stays. The token is the first index whose running sum of kept weights exceeds
    ``u`` times their total; ``temperature`` 0 takes the largest logit. Each setting is a number
    or a ``[B]`` tensor (fp32; ``top_k`` int32). A row gives the same token in every batch."""
    per_row = [t for t in (temperature, top_k, top_p, min_p) if isinstance(t, torch.Tensor)]
    dev = _on_one_device(logits, u, *per_row)
    if logits.dim() != 2:
        raise ValueError("logits must be [B, V]")
    B, V = logits.shape
    _want(u, "u", torch.float32, (B,))
    f32, inf = torch.float32, float("inf")
    t, tv = _setting(temperature, "temperature", B, f32, 0.0, 3e38)
    k, kv = _setting(top_k, "top_k", B, torch.int32, 0, 2**31 - 1)
    p, pv = _setting(top_p, "top_p", B, f32, 0.0, inf)
    mp, mv = _setting(min_p, "min_p", B, f32, 0.0, 1.0)
    if V > 1 and logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()  # also of a row given to all by expand
    token = torch.empty(B, dtype=torch.int64, device=dev)
    logprob = torch.empty(B, dtype=f32, device=dev) if return_logprob else None
    _run(dev, "dsalt_sample", logits.data_ptr(), _dt(logits), B, V, logits.stride(0) if B > 1 else V, u.data_ptr(),
         _ptr(t), tv, _ptr(k), kv, _ptr(p), pv, _ptr(mp), mv, token.data_ptr(), _ptr(logprob))
    return (token, logprob) if return_logprob else token


# --------------------------------------------------------------------------- a decoder stack's state
class PagedCache:
    """Keys and values of ``max_seqs`` sequences for ``n_layers`` layers in pages of
    ``page_size`` tokens, with what the landmark selection needs of them (norms and widths per
    position) and the current landmark sets ``[H, max_seqs, k]`` per layer.

    Rows are sequences, which begin and end on their own: :meth:`reserve` takes the number of
    new tokens of each row, 0 among them, and what follows (:meth:`append`, :meth:`attention`)
    packs the tokens of the rows that have some. ``lens`` is the host's copy of the lengths, kept
    so that block borders are known without reading the device; a row whose tokens the pool or
    the tables cannot hold is refused here, before anything is launched. The norms and widths are
    not paged: ``8 + 4 n_kv_heads`` bytes per layer, row and position of ``max_len``."""

    def __init__(self, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, k_lmk: int, *, max_seqs: int,
                 max_len: int, n_pages: int | None = None, page_size: int = 64, device="cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if head_dim not in HEAD_SIZES:
            raise ValueError(f"head size {head_dim}: the cache holds heads of {' or '.join(map(str, HEAD_SIZES))}")
        if n_kv_heads < 1 or n_heads % n_kv_heads:
            raise ValueError(f"n_heads ({n_heads}) must be a multiple of n_kv_heads ({n_kv_heads})")
        if not 1 <= max_seqs <= MAX_ROWS or not 1 <= max_len <= MAX_POSITIONS - page_size:
            raise ValueError(f"max_seqs must be in [1, {MAX_ROWS}] and max_len in [1, {MAX_POSITIONS - page_size}]")
        self.max_seqs, self.max_len, self.page_size = max_seqs, max_len, page_size
        self.max_pages = -(-max_len // page_size)
        self.n_pages = self.max_pages * max_seqs if n_pages is None else int(n_pages)
        if not 0 <= self.n_pages * n_kv_heads * page_size <= MAX_POSITIONS:
            raise ValueError(f"a pool of {self.n_pages} pages: it holds {MAX_POSITIONS} positions of all kv heads at most")
        dev = torch.device(device)
        i32 = torch.int32
        self.block_tables = torch.full((max_seqs, self.max_pages), -1, dtype=i32, device=dev)
        self.seq_lens = torch.zeros(max_seqs, dtype=i32, device=dev)
        self.free_pages = torch.arange(self.n_pages - 1, -1, -1, dtype=i32, device=dev)
        self.n_free = torch.full((1,), self.n_pages, dtype=i32, device=dev)
        self.lens = [0] * max_seqs
        kv = (n_layers, self.n_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.zeros(kv, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.v = torch.zeros(kv, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.k_scale = torch.zeros(n_layers, self.n_pages, n_kv_heads, device=dev)
        self.v_scale = torch.zeros(n_layers, self.n_pages, n_kv_heads, device=dev)
        self.xnorm = torch.zeros(n_layers, max_seqs, max_len, device=dev)
        self.vnorm = torch.zeros(n_layers, max_seqs, max_len, n_kv_heads, device=dev)
        self.width = torch.zeros(n_layers, max_seqs, max_len, dtype=i32, device=dev)
        self.lmk = torch.full((n_layers, n_heads, max_seqs, k_lmk), -1, dtype=i32, device=dev)
        self._rows = self._cu_new = None  # of the tokens reserved last: each one's row, each row's first
        self._new_lens = [0] * max_seqs
        self._block_of = [[-1] * max_seqs for _ in range(n_layers)]  # whose set `lmk` holds

    def pages_held(self) -> int:
        return sum(-(-n // self.page_size) for n in self.lens)

    def reserve(self, new_lens) -> SlotPlan:
        """Slots for ``new_lens`` (a list, one number per row) more tokens, packed row after row."""
        new_lens = [int(n) for n in new_lens]
        if len(new_lens) != self.max_seqs or min(new_lens) < 0:
            raise ValueError(f"new_lens must give {self.max_seqs} numbers of new tokens")
        lens = [a + b for a, b in zip(self.lens, new_lens)]
        if max(lens) > self.max_len:
            raise ValueError(f"a sequence of {max(lens)} tokens in a cache for {self.max_len}")
        need = sum(-(-n // self.page_size) for n in lens)
        if need > self.n_pages:
            raise ValueError(f"{need} pages wanted of a pool of {self.n_pages}")
        dev = self.seq_lens.device
        new = torch.tensor(new_lens, dtype=torch.int32, device=dev)
        plan = reserve_slots(self.block_tables, self.seq_lens, new, self.free_pages, self.n_free, self.page_size,
                             sum(new_lens), inplace=True)
        self.lens = lens
        self._rows = torch.repeat_interleave(torch.arange(self.max_seqs, device=dev), new.long(),
                                             output_size=sum(new_lens))
        self._cu_new, self._new_lens = plan.cu_new, new_lens
        return plan

    def pick(self, x):
        """The lines of ``x [max_seqs, ...]`` of the rows that got tokens last, packed."""
        rows = [r for r, n in enumerate(self._new_lens) if n]
        return x if len(rows) == self.max_seqs else x[torch.tensor(rows, device=x.device)]

    def spread(self, x):
        """The reverse: ``x``, a line for each row that got tokens last, as ``[max_seqs, ...]`` with
        zeros for the other rows."""
        rows = [r for r, n in enumerate(self._new_lens) if n]
        if len(rows) == self.max_seqs:
            return x
        return x.new_zeros(self.max_seqs, *x.shape[1:]).index_copy_(0, torch.tensor(rows, device=x.device), x)

    def release(self, rows) -> None:
        """Ends the sequences of these rows; their pages go back to the pool."""
        rows = [int(r) for r in rows]
        if any(not 0 <= r < self.max_seqs for r in rows):
            raise ValueError(f"rows must lie in [0, {self.max_seqs})")
        flags = [False] * self.max_seqs
        for r in rows:
            flags[r] = True
            self.lens[r] = 0
            for blocks in self._block_of:
                blocks[r] = -1
        release_slots(self.block_tables, self.seq_lens, torch.tensor(flags, device=self.seq_lens.device), self.free_pages,
                      self.n_free, self.page_size)

    def append(self, layer: int, k, v, w, xn, vn, plan: SlotPlan) -> None:
        """New tokens of all rows (packed as ``plan`` says) into one layer."""
        append_cache(k, v, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], plan.slots)
        at = (self._rows, plan.positions.long())
        self.xnorm[layer].index_put_(at, xn)
        self.vnorm[layer].index_put_(at, vn)
        self.width[layer].index_put_(at, w)

    def update_landmarks(self, layer: int, alpha, k_lmk: int, block: int) -> None:
        """The set of the block that each row's last position lies in, where it is a new one: drawn
        from the positions before the block, with their statistics, as
        :func:`dsalt_b200.ops.select_landmarks` does in block-causal mode."""
        H = self.lmk.shape[1]
        for r, n in enumerate(self.lens):
            b = (n - 1) // block
            if n == 0 or k_lmk == 0 or self._block_of[layer][r] == b:
                continue
            self._block_of[layer][r] = b
            if b == 0:
                self.lmk[layer, :, r] = -1
                continue
            end = b * block + 1
            with torch.cuda.device(self.lmk.device):
                sets = ops.select_block_range(self.xnorm[layer, r, :end], self.vnorm[layer, r, :end],
                                              self.width[layer, r, :end], alpha, k_lmk, H, block, b, b + 1)
            self.lmk[layer, :, r] = sets[:, 0]

    def attention(self, layer: int, q, w):
        """One query token for each row that got one last (packed: rows without are passed over) over
        one layer."""
        if max(self._new_lens) > 1:  # the landmark sets are those of each row's last position
            raise ValueError("attention takes one query token per row")
        lmk = self.lmk[layer] if self.lmk.shape[-1] > 0 else None
        return cache_attention(q.contiguous(), self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                               self.block_tables, self.seq_lens, cu_q=None if min(self._new_lens) else self._cu_new,
                               w_sizes=w, lmk_indices=lmk)
