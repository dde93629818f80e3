"""Attention of single tokens over a paged cache.

Each row of the batch attends over the tokens of one sequence of a
``PagedKVCache`` (or of tensors laid out like its pages).  Rows that begin
with the same pages, because they were forked from one sequence or admitted
behind one system prompt, can say so with ``SharedPrefix``: their common pages
are then read once for all of them.

On the GPU this is ``ops/csrc/paged_attention.hip`` (bf16 and fp16, head sizes
64 and 128); on the CPU a plain computation in 32 bits or more.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from .paged_kv_cache import MOST_TOKENS
from ... import ops as _ops

HEAD_SIZES = (64, 128)


@dataclass
class SharedPrefix:
    """Which rows of the batch begin with the same pages.

    Rows ``rows[g]`` to ``rows[g + 1]`` (int32 [groups + 1] on the device,
    ascending) share their first ``lengths[g]`` tokens (int32 [groups]; whole
    pages count, a rest is left to each row): the page tables of these rows
    name the same pages there, as far as each row is long, which is not looked
    at again; one that holds all of them is read for all.  Rows outside every
    group share nothing.  ``max_rows`` and ``max_length`` are what the host
    knows about the largest group; they choose how the work is cut, not what
    is computed.
    """

    rows: torch.Tensor
    lengths: torch.Tensor
    max_rows: int
    max_length: int


def paged_attention_supported(query: torch.Tensor) -> bool:
    """Whether the GPU kernels take this query."""
    return (query.is_cuda and _ops.have_ops()
            and query.dtype in (torch.bfloat16, torch.float16)
            and query.shape[-1] in HEAD_SIZES)


def _paged_attention_plain(q, k, v, tables, lengths, slots, scale):
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    b, nh, d = q.shape
    pages, ng, page = k.shape[:3]
    out = torch.zeros(b, nh, d, dtype=wide, device=q.device)
    for i, s in enumerate(range(b) if slots is None else slots.tolist()):
        if not 0 <= s < lengths.shape[0]:
            continue
        n = max(0, min(int(lengths[s]), tables.shape[1] * page))
        if n == 0:
            continue
        ids = tables[s, :-(-n // page)].long()
        fine = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:n]
        ids = ids.clamp(0, pages - 1)

        def tokens(x):      # [n, ng, d] -> [ng, tokens, d]
            x = x[ids].transpose(1, 2).reshape(-1, ng, d)[:n][fine]
            return x.transpose(0, 1).to(wide)

        if not bool(fine.any()):
            continue
        s_ = torch.matmul(q[i].to(wide).view(ng, nh // ng, d),
                          tokens(k).transpose(1, 2)) * scale
        out[i] = torch.matmul(torch.softmax(s_, -1),
                              tokens(v)).reshape(nh, d)
    return out.to(q.dtype)


def _check(query, key_pages, value_pages, page_tables, lengths, slots,
           shared_prefix, scale):
    """What the GPU's entry checks, for the CPU."""
    if query.dim() != 3 or key_pages.dim() != 4 or \
            value_pages.shape != key_pages.shape:
        raise ValueError("paged_attention: query must be [b, heads, d], key "
                         "and value pages [P, groups, page, d]")
    if key_pages.shape[3] != query.shape[2] or key_pages.shape[1] < 1 or \
            query.shape[1] % key_pages.shape[1] or key_pages.shape[0] < 1:
        raise ValueError(
            f"paged_attention: query {tuple(query.shape)} and pages "
            f"{tuple(key_pages.shape)} do not fit each other")
    page = key_pages.shape[2]
    if page < 16 or page % 16:
        raise ValueError("paged_attention: pages must hold a multiple of 16 "
                         "tokens")
    if key_pages.dtype != query.dtype or value_pages.dtype != query.dtype or \
            not query.is_floating_point():
        raise ValueError("paged_attention: query and pages must share one "
                         "floating type")
    ints = [("page_tables", page_tables, 2), ("lengths", lengths, 1)]
    if slots is not None:
        ints.append(("slots", slots, 1))
    if shared_prefix is not None:
        ints += [("shared_prefix.rows", shared_prefix.rows, 1),
                 ("shared_prefix.lengths", shared_prefix.lengths, 1)]
        if shared_prefix.rows.numel() != shared_prefix.lengths.numel() + 1:
            raise ValueError("paged_attention: shared_prefix.rows must be "
                             "one longer than its lengths")
    for name, t, dim in ints:
        if t.dim() != dim or t.dtype != torch.int32:
            raise ValueError(f"paged_attention: {name} must be an int32 "
                             f"tensor of {dim} dimension(s)")
    if any(t.device != query.device for t in
           [key_pages, value_pages] + [t for _, t, _ in ints]):
        raise ValueError("paged_attention: all tensors must be on the "
                         "query's device")
    if lengths.shape[0] != page_tables.shape[0] or \
            page_tables.shape[0] < 1 or page_tables.shape[1] < 1 or \
            (slots if slots is not None else lengths).shape[0] != \
            query.shape[0]:
        raise ValueError("paged_attention: one length for each table, one "
                         "table or slot for each row")
    if page_tables.shape[1] * page > MOST_TOKENS:
        raise ValueError("paged_attention: tables of 2^31 tokens, or 8191 "
                         "fewer, are too long")
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("paged_attention: softmax_scale must be positive "
                         "and finite")


def paged_attention(query: torch.Tensor, key_pages: torch.Tensor,
                    value_pages: torch.Tensor, page_tables: torch.Tensor,
                    lengths: torch.Tensor,
                    slots: Optional[torch.Tensor] = None,
                    shared_prefix: Optional[SharedPrefix] = None,
                    softmax_scale: Optional[float] = None,
                    max_length: Optional[int] = None) -> torch.Tensor:
    """query [b, heads, d] over key_pages and value_pages [P, groups, page,
    d]; returns [b, heads, d].

    Row i sees the first lengths[s] tokens of the pages page_tables[s], with
    s = slots[i], or i without slots (int32, all on the query's device).
    ``max_length`` is what the host knows about the longest row (by default
    all that a table can hold); it chooses how the work is cut, not what is
    computed.  A row of no tokens gives zeros; so does a slot out of range,
    and a page number out of the pool leaves its tokens out."""
    if torch.is_grad_enabled() and (query.requires_grad
                                    or key_pages.requires_grad
                                    or value_pages.requires_grad):
        raise ValueError("paged_attention: has no gradient; call it under "
                         "torch.no_grad()")
    if query.is_cuda:
        rows = shared = None
        max_rows = max_prefix = 0
        if shared_prefix is not None:
            rows, shared = shared_prefix.rows, shared_prefix.lengths
            max_rows = shared_prefix.max_rows
            max_prefix = shared_prefix.max_length
        return _ops.get_ops().paged_attn(
            query, key_pages, value_pages, page_tables, lengths, slots,
            max_length, rows, shared, max_rows, max_prefix, softmax_scale)
    scale = (1.0 / math.sqrt(query.shape[-1]) if softmax_scale is None
             else float(softmax_scale))
    _check(query, key_pages, value_pages, page_tables, lengths, slots,
           shared_prefix, scale)
    if any(forward_ad.unpack_dual(x).tangent is not None
           for x in (query, key_pages, value_pages)):
        raise ValueError("paged_attention: has no gradient, in forward mode "
                         "neither")
    return _paged_attention_plain(query, key_pages, value_pages, page_tables,
                                  lengths, slots, scale)
