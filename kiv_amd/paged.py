"""Paged key/value cache: ragged batches of sequences of different lengths.

The tiered cache grows one window for a whole batch; sequences that come, go
and grow on their own are held here instead.  :class:`PagedKVCache` is one
layer's pool of pages, :class:`PagedBatch` the new tokens of a step (packed
one sequence behind the other, with each sequence's length and block table;
built once a step and used for every layer), :func:`paged_append` writes the
new keys and values to their pages with head norms and position rotation on
the way, and :func:`paged_attention` attends over the pages: chunks of new
tokens, single tokens, or both in one batch.

Lengths and tables are read on the device only, so nothing here synchronises
and a captured HIP graph follows what the arrays hold at each replay.  No
counterpart in the reference.
"""

from __future__ import annotations

import torch

from . import _native as nat
from .rotary import HeadNorm, Rotary, aligned_rows, no_grad_check, out_rows


class PagedKVCache:
    """A pool of ``num_pages`` pages of ``page_size`` tokens of one layer's K and V.

    ``k`` and ``v`` are [num_pages, num_kv_heads, page_size, head_dim] views;
    with ``tokens_first`` a token's heads lie together in memory (head-major
    pages otherwise).  The rows are uninitialised until appended.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                 tokens_first: bool = False) -> None:
        if min(num_pages, page_size, num_kv_heads, head_dim) < 1:
            raise ValueError("num_pages, page_size, num_kv_heads and head_dim must be >= 1")
        nat.dtype_code(dtype)
        shape = ((num_pages, page_size, num_kv_heads, head_dim) if tokens_first
                 else (num_pages, num_kv_heads, page_size, head_dim))
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self._bind(*(t.transpose(1, 2) if tokens_first else t for t in (k, v)))

    @classmethod
    def from_pages(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKVCache":
        """A cache over existing [num_pages, num_kv_heads, page_size, head_dim]
        tensors of equal shape, strides and dtype (any strides with unit
        stride over head_dim)."""
        self = cls.__new__(cls)
        self._bind(k, v)
        return self

    def _bind(self, k: torch.Tensor, v: torch.Tensor) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("K and V pages must be equal [num_pages, num_kv_heads, page_size, head_dim] tensors")
        if min(k.shape) < 1:
            raise ValueError(f"empty pages {tuple(k.shape)}")
        nat.check_sizes("PagedKVCache", *k.shape)
        if k.stride() != v.stride():
            raise ValueError("K and V pages must have the same strides")
        if not k.is_cuda:
            raise ValueError("the paged cache lives on a GPU")
        out_rows(k, k, "K pages")
        out_rows(v, v, "V pages")
        self._k, self._v = k, v
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._args = nat.PagedCacheArgs(k.data_ptr(), v.data_ptr(), nat.layout(k).strides, self.num_pages,
                                        self.page_size, self.num_kv_heads, self.head_dim, nat.dtype_code(k.dtype), 0)
        self._geometry = (tuple(k.shape), k.stride(), k.dtype)

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    def memory_bytes(self) -> int:
        """Bytes of the pool's K and V rows."""
        return 2 * self._k.numel() * self._k.element_size()


class PagedBatch:
    """The new tokens of one step, and the caches' sequences they belong to.

    block_table  [S, W] int32: the pages of each sequence in order; entries
                 outside the pool (-1, say) are pages that are not there.
    kv_len       [S] int32: keys of each sequence, the new tokens' among them.
    cu_q         [S + 1] int32: first packed row of each sequence and the end
                 of the last; rows past it are no sequence's.  None: one new
                 token a sequence.
    max_q_len, max_kv_len  bounds of the lengths, known to the host; they
                 choose the kernel only, and with it the results' rounding
                 (a wrong one costs time).  Defaults: no bound.

    The arrays stay the caller's: update them in place between steps (or
    between replays of a captured graph).
    """

    def __init__(self, block_table: torch.Tensor, kv_len: torch.Tensor, cu_q: torch.Tensor | None = None,
                 max_q_len: int | None = None, max_kv_len: int | None = None) -> None:
        if block_table.dim() != 2 or kv_len.dim() != 1:
            raise ValueError("block_table must be [S, W] and kv_len [S]")
        for name, n in (("max_q_len", max_q_len), ("max_kv_len", max_kv_len)):
            if n is not None and n < 0:
                raise ValueError(f"{name} must not be negative, got {n}")
        S, W = block_table.shape
        nat.check_sizes("PagedBatch", S, W)
        if cu_q is None:
            cu_q = torch.arange(S + 1, dtype=torch.int32, device=block_table.device)
            max_q_len = 1
        if kv_len.shape[0] != S or cu_q.dim() != 1 or cu_q.shape[0] != S + 1:
            raise ValueError(f"block_table has {S} sequences, kv_len {tuple(kv_len.shape)}, cu_q {tuple(cu_q.shape)}")
        for name, t in (("block_table", block_table), ("kv_len", kv_len), ("cu_q", cu_q)):
            if t.dtype != torch.int32:
                raise TypeError(f"{name} must be int32, not {t.dtype}")
            if not t.is_cuda or t.device != block_table.device:
                raise ValueError(f"{name} must be on the batch's GPU")
            if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{name} must have unit stride")
        self._block_table, self._kv_len, self._cu_q = block_table, kv_len, cu_q
        self.num_seqs, self.device = S, block_table.device
        big = 2**31 - 1
        self._args = nat.PagedBatchArgs(
            cu_q.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(), block_table.stride(0) if S > 1 else 0, S, W, 0,
            big if max_q_len is None else min(max_q_len, big), big if max_kv_len is None else min(max_kv_len, big), 0)
        self._geometry = (S, W, self._args.max_q_len, self._args.max_kv_len, self.device)

    @property
    def block_table(self) -> torch.Tensor:
        return self._block_table

    @property
    def kv_len(self) -> torch.Tensor:
        return self._kv_len

    @property
    def cu_q(self) -> torch.Tensor:
        return self._cu_q


def _packed_layout(t: torch.Tensor, name: str, cache: PagedKVCache, heads: int | None) -> nat.Layout:
    """Layout of packed rows [tokens, heads, head_dim] that go with the cache."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {heads or 'heads'}, {cache.head_dim}], got {tuple(shape)}")
    nat.check_sizes(name, *shape)
    if t.dtype != cache.dtype:
        raise TypeError(f"{name} is {t.dtype}, the cache {cache.dtype}")
    return nat.layout(t)


def paged_append(cache: PagedKVCache, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor,
                 q: torch.Tensor | None = None, positions: torch.Tensor | None = None, rotary: Rotary | None = None,
                 q_norm: HeadNorm | None = None, k_norm: HeadNorm | None = None, v_norm: HeadNorm | None = None,
                 q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write the batch's new K and V rows [tokens, Hkv, D] to their pages.

    Token r of sequence b goes to key index kv_len[b] - cu_q[b + 1] + r
    (kv_len counts the new tokens), K normed (``k_norm``) and turned
    (``rotary``) on the way, V normed (``v_norm``) or copied.  positions:
    [tokens] or, with ``rotary.axes``, [axes, tokens]; None turns each token
    by its key index.  With q [tokens, Hq, D] the queries are normed
    (``q_norm``) and turned in the same launch, into ``q_out`` (new by
    default; may be q itself); returns it, else None.  Any other overlap of the
    pages or ``q_out`` with each other or the inputs is refused.  Rows past the
    last sequence are left alone, in the pages and in ``q_out``; a token whose
    page is not there is dropped; a slot that two new tokens name holds parts
    of both rows.
    """
    no_grad_check("paged_append", q, k, v, cache._k, cache._v)
    key = (cache._geometry, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype,
           None if q is None else (q.shape, q.stride(), q.dtype))
    plan = _append_plans.get(key)
    if plan is None:
        plan = nat.remember(_append_plans, key, _append_plan(cache, k, v, q))
    template, T, copy = plan
    dev, D = cache.device, cache.head_dim
    if k.device != dev or v.device != dev or batch.device != dev or (q is not None and q.device != dev):
        raise ValueError(f"k, v, q, the batch and the cache must be on one device ({dev})")
    args = nat.PagedAppendArgs.from_buffer_copy(template)
    args.cache, args.batch = cache._args, batch._args
    args.batch.total_q = T
    at, vat = k.data_ptr(), v.data_ptr()
    if copy or (at | vat) & 15:
        k, at, lay = aligned_rows(k)
        args.k_stride = lay.strides
        v, vat, lay = aligned_rows(v)
        args.v_stride = lay.strides
    args.k, args.v = at, vat
    if q is not None:
        at = q.data_ptr()
        if copy or at & 15:
            q, at, lay = aligned_rows(q)
            args.q_stride = lay.strides
            args.q_out_stride = nat.layout(torch.empty_like(q, device="meta")).strides
        args.q = at
        if q_out is None:
            q_out = torch.empty_like(q)
            args.q_out = q_out.data_ptr()
        else:
            no_grad_check("paged_append", q_out)
            args.q_out, lay = out_rows(q_out, q, "q_out")
            args.q_out_stride = lay.strides
        if q_norm is not None:
            args.q_norm = q_norm.check(D, dev)
    elif q_norm is not None or q_out is not None:
        raise ValueError("q_norm and q_out need q")
    if k_norm is not None:
        args.k_norm = k_norm.check(D, dev)
    if v_norm is not None:
        args.v_norm = v_norm.check(D, dev)
    if rotary is not None:
        args.rotary = rotary._args
        rotary.fill(args.rotary, positions, 1, T, dev, False)
    elif positions is not None:
        raise ValueError("positions need a rotation")
    nat.call("kiv_paged_append", args, dev)
    return q_out


_append_plans: dict[tuple, tuple] = {}


def _append_plan(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None) -> tuple:
    """What a call's shapes, strides and dtypes give: (its arguments without
    addresses, tokens, whether rows must be copied)."""
    args = nat.PagedAppendArgs()
    kl, vl = _packed_layout(k, "k", cache, cache.num_kv_heads), _packed_layout(v, "v", cache, cache.num_kv_heads)
    args.k_stride, args.v_stride = kl.strides, vl.strides
    T, copy = k.shape[0], not (kl.chunked and vl.chunked)
    if v.shape[0] != T:
        raise ValueError(f"k has {T} tokens, v {v.shape[0]}")
    if q is not None:
        ql = _packed_layout(q, "q", cache, None)
        if q.shape[0] != T:
            raise ValueError(f"k has {T} tokens, q {q.shape[0]}")
        args.num_q_heads, args.q_stride = q.shape[1], ql.strides
        args.q_out_stride = nat.layout(torch.empty_like(q, device="meta")).strides
        copy = copy or not ql.chunked
    return args, T, copy


def paged_attention(query: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, scaling: float, window: int = 0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q K^T * scaling) V of the batch's packed rows [tokens, Hq, D]
    over the keys of their sequences, up to each token's own
    (kv_len[b] - cu_q[b + 1] + row); with ``window`` the last ``window`` of
    those.  Append the new tokens first.  Query head h reads key head
    h // (Hq / Hkv); head_dim 32, 64, 96, 128, 192 or 256.  fp32 inside; fp16
    and bf16 batches of more than 16 rows a key head and sequence (by the
    batch's max_q_len) weight V by probabilities rounded to the dtype.

    Returns [tokens, Hq, D]: ``out`` (contiguous; refused if it overlaps the
    query or the pages) or a new tensor.  Rows that see no key are zero; rows
    past the last sequence stay as they are (in a new tensor: undefined).
    """
    no_grad_check("paged_attention", query, cache._k, cache._v)
    dev = cache.device
    if query.device != dev or batch.device != dev:
        raise ValueError(f"query is on {query.device}, the batch on {batch.device}, the cache on {dev}")
    key = (query.shape, query.stride(), query.dtype, window, cache._geometry, batch._geometry)
    plan = _attention_plans.get(key)
    if plan is None:
        plan = nat.remember(_attention_plans, key, _attention_plan(query, cache, batch, window))
    template, need, T, copy = plan
    args = nat.PagedAttentionArgs.from_buffer_copy(template)
    args.cache, args.batch = cache._args, batch._args
    args.batch.total_q = T
    q, at = query, query.data_ptr()
    if copy or at & 15:
        q, at, lay = aligned_rows(query)
        args.q_stride = lay.strides
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        no_grad_check("paged_attention", out)
        out_rows(out, query, "out")
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    args.q, args.out, args.scaling = at, out.data_ptr(), scaling
    if need:
        # Scratch of this call, from torch's allocator on the current stream:
        # calls on other streams, and captured graphs, have their own.
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    nat.call("kiv_paged_attention", args, dev)
    return out


_attention_plans: dict[tuple, tuple] = {}


def _attention_plan(query: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, window: int) -> tuple:
    """What a call's shapes, strides, dtypes and bounds give: (its arguments
    without addresses, workspace bytes, tokens, whether the query must be
    copied)."""
    lay = _packed_layout(query, "query", cache, None)
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    args = nat.PagedAttentionArgs()
    args.cache, args.batch = cache._args, batch._args
    args.batch.total_q, args.num_q_heads = query.shape[0], query.shape[1]
    args.q_stride, args.window, args.scaling = lay.strides, min(window, 2**31 - 1), 1.0
    with torch.cuda.device(cache.device):
        need = nat.lib().kiv_paged_attention_workspace_size(args)
    return args, need, query.shape[0], not lay.chunked
