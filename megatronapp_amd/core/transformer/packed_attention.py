"""Attention over packed sequences of different lengths, with its gradient.

A stream holds sequences one behind the other; ``PackedSeqParams`` says where
each begins.  Queries may be fewer than keys (a prompt continued from a
cache): the last query sees the last key.  Rows that see no key, and rows
before the first or behind the last sequence, give zeros, and get and give no
gradient.

On the GPU this is ``ops/csrc/packed_attention.hip`` (bf16 and fp16, head
sizes 64 and 128), whose gradient cannot be differentiated again, and which
refuses forward-mode derivatives; on the CPU a plain computation in 32 bits or
more.  A sequence's values reach no other sequence, whatever they are.  Within
one, what is not finite may reach rows of the same tile that do not see it
(nothing times NaN is NaN): from v earlier rows, and in the gradients from k,
from q and from the output's gradient too.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from ..packed_seq_params import PackedSeqParams
from ... import ops as _ops

HEAD_SIZES = (64, 128)


def packed_attention_supported(query: torch.Tensor) -> bool:
    """Whether the GPU kernels take this query."""
    return (query.is_cuda and _ops.have_ops()
            and query.dtype in (torch.bfloat16, torch.float16)
            and query.shape[-1] in HEAD_SIZES)


def _check(query, key, value, cu_q, cu_k, scale):
    """What the GPU's entry checks, for the CPU."""
    if query.dim() not in (3, 4) or key.dim() != query.dim() \
            or value.shape != key.shape:
        raise ValueError(
            "packed_attention: query, key, value must be [t, heads, hn] or "
            f"[t, b, heads, hn], got {tuple(query.shape)}, "
            f"{tuple(key.shape)}, {tuple(value.shape)}")
    if key.shape[-1] != query.shape[-1] or key.shape[-2] < 1 or \
            query.shape[-2] % key.shape[-2] or \
            key.shape[1:-2] != query.shape[1:-2]:
        raise ValueError(
            f"packed_attention: query {tuple(query.shape)} and key "
            f"{tuple(key.shape)} do not fit each other")
    if key.dtype != query.dtype or value.dtype != query.dtype or \
            not query.is_floating_point():
        raise ValueError("packed_attention: query, key and value must share "
                         "one floating type")
    if key.device != query.device or value.device != query.device:
        raise ValueError("packed_attention: query, key and value must be on "
                         "one device")
    for cu in (cu_q, cu_k):
        if cu.dim() != 1 or cu.numel() < 1 or cu.shape != cu_q.shape or \
                cu.dtype not in (torch.int32, torch.int64):
            raise ValueError("packed_attention: cu_seqlens must be int32 or "
                             "int64 [sequences + 1], the same for both")
        if cu.device != query.device:
            raise ValueError("packed_attention: cu_seqlens must be on the "
                             "query's device")
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("packed_attention: softmax_scale must be positive "
                         "and finite")


def _spans(cu, total):
    """Begins and ends of the sequences, kept within the stream."""
    begins, ends = [], []
    for a, b in zip(cu[:-1], cu[1:]):
        a = max(0, min(a, total))
        begins.append(a)
        ends.append(max(a, min(b, total)))
    return begins, ends


def _packed_attention_plain(q, k, v, cu_q, cu_k, scale, causal):
    """[t, b, h, d] in 32 bits or more, one sequence at a time."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    rep = q.shape[2] // k.shape[2]
    out = torch.zeros(q.shape, dtype=wide, device=q.device)
    for qa, qb, ka, kb in zip(*_spans(cu_q.tolist(), q.shape[0]),
                              *_spans(cu_k.tolist(), k.shape[0])):
        if qa == qb or ka == kb:
            continue
        x = q[qa:qb].to(wide).permute(1, 2, 0, 3)
        y = k[ka:kb].to(wide).permute(1, 2, 3, 0).repeat_interleave(rep, 1)
        z = v[ka:kb].to(wide).permute(1, 2, 0, 3).repeat_interleave(rep, 1)
        s = torch.matmul(x, y) * scale
        if causal:
            sq, sk = qb - qa, kb - ka
            place = torch.arange(sq, device=q.device)[:, None] + sk - sq
            hide = torch.arange(sk, device=q.device)[None] > place
            s = s.masked_fill(hide, -math.inf)
            # a row without keys: any finite score, and no weight
            s = s.masked_fill(hide.all(-1, keepdim=True), 0.0)
            p = torch.softmax(s, -1).masked_fill(hide, 0.0)
        else:
            p = torch.softmax(s, -1)
        out = out.index_copy(0, torch.arange(qa, qb, device=q.device),
                             torch.matmul(p, z).permute(2, 0, 1, 3))
    return out.to(q.dtype)


def packed_attention(query: torch.Tensor, key: torch.Tensor,
                     value: torch.Tensor, packed_seq_params: PackedSeqParams,
                     softmax_scale: Optional[float] = None,
                     causal: bool = True) -> torch.Tensor:
    """query [t, np, hn] or [t, b, np, hn], key and value the same with ng
    heads that divide np (and a length of their own); returns the query's
    shape.  ``cu_seqlens_kv`` defaults to ``cu_seqlens_q``; both ascend, are
    given on the query's device, and are not read by the host there, so ends
    that run out of the stream are cut off at it rather than refused."""
    cu_q = packed_seq_params.cu_seqlens_q
    cu_k = packed_seq_params.cu_seqlens_kv
    if cu_q is None:
        raise ValueError("packed_attention: cu_seqlens_q is missing")
    if query.is_cuda:
        return _ops.get_ops().packed_attention(query, key, value, cu_q, cu_k,
                                               softmax_scale, causal)
    cu_k = cu_q if cu_k is None else cu_k
    scale = (1.0 / math.sqrt(query.shape[-1]) if softmax_scale is None
             else float(softmax_scale))
    _check(query, key, value, cu_q, cu_k, scale)
    flat = query.dim() == 3
    if flat:
        query, key, value = (x.unsqueeze(1) for x in (query, key, value))
    out = _packed_attention_plain(query, key, value, cu_q, cu_k, scale,
                                  causal)
    return out.squeeze(1) if flat else out
