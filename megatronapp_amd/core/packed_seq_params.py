"""Packed-sequence metadata (reference core/packed_seq_params.py).

Multiple variable-length sequences packed into one token stream; the
cu_seqlens prefix arrays mark boundaries.  FlashAttention hands them to the
packed kernels; DotProductAttention turns them into a block-diagonal mask, so
that tokens never attend across sequence boundaries either way.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch


@dataclass
class PackedSeqParams:
    qkv_format: str = "thd"
    cu_seqlens_q: Optional[torch.Tensor] = None
    cu_seqlens_kv: Optional[torch.Tensor] = None
    max_seqlen_q: Optional[int] = None
    max_seqlen_kv: Optional[int] = None


def _sequences(cu_seqlens: torch.Tensor, total: int):
    """Each place's sequence, n before the first one and behind the last, and
    the sequences' begins and ends, kept within the stream."""
    cu = cu_seqlens.long().clamp(0, total)
    place = torch.arange(total, device=cu.device)
    n = cu.numel() - 1
    seq = torch.searchsorted(cu[1:].contiguous(), place, right=True)
    return torch.where(place < cu[0], n, seq), place, cu


def packed_attention_mask(cu_seqlens: torch.Tensor, total: int,
                          causal: bool = True,
                          cu_seqlens_kv: Optional[torch.Tensor] = None,
                          total_kv: Optional[int] = None) -> torch.Tensor:
    """[1, 1, total, total_kv] bool mask, True = masked: block-diagonal over
    the packed segments, causal within each (a segment's last query sees its
    last key).  Places outside all segments see nothing and are not seen."""
    seq_q, place_q, cu_q = _sequences(cu_seqlens, total)
    if cu_seqlens_kv is None and total_kv is None:
        seq_k, place_k, cu_k = seq_q, place_q, cu_q
    else:
        seq_k, place_k, cu_k = _sequences(
            cu_seqlens if cu_seqlens_kv is None else cu_seqlens_kv,
            total if total_kv is None else total_kv)
    n = cu_q.numel() - 1
    mask = (seq_q[:, None] != seq_k) | (seq_q[:, None] == n)
    if causal and n:
        # how many places in front of its segment's end each one lies
        behind_q = cu_q[1:][seq_q.clamp(max=n - 1)] - place_q
        behind_k = cu_k[1:][seq_k.clamp(max=n - 1)] - place_k
        mask |= behind_q[:, None] > behind_k
    return mask.view(1, 1, mask.shape[0], mask.shape[1])
