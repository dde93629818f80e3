"""Inference context of the dynamic engine over a paged cache.

Takes the place of :class:`DynamicInferenceContext` where the engine is given
a page size.  Prompts that are admitted together run as one packed stream
(``packed_attention``), each decode step reads the pages of all running
sequences where they lie (``paged_attention``), and sequences that were forked
from one prompt share its pages, which a step then reads once.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from .. import parallel_state
from ..packed_seq_params import PackedSeqParams, packed_attention_mask
from ..transformer.packed_attention import packed_attention
from .paged_attention import HEAD_SIZES, SharedPrefix, paged_attention
from .paged_kv_cache import PagedKVCache


class PagedInferenceContext:
    is_paged = True
    is_dynamic = False
    is_graph_context = False

    def __init__(self, num_layers: int, num_query_groups: int, head_dim: int,
                 max_slots: int, max_sequence_length: int,
                 page_size: int = 64, num_pages: Optional[int] = None,
                 dtype=torch.bfloat16, device="cuda"):
        if torch.device(device).type == "cuda" and (
                dtype not in (torch.bfloat16, torch.float16)
                or head_dim not in HEAD_SIZES):
            raise ValueError(
                "PagedInferenceContext: on the GPU bf16 or fp16 with head "
                f"size 64 or 128, got {dtype}, {head_dim}")
        per_slot = -(-max_sequence_length // page_size)
        self.cache = PagedKVCache(
            num_layers, num_pages or max_slots * per_slot, page_size,
            num_query_groups, head_dim, max_slots, max_sequence_length,
            dtype=dtype, device=device)
        self.max_slots = max_slots
        self.max_sequence_length = max_sequence_length
        self.sequence_len_offset = 0
        self.host_lengths = [0] * max_slots
        self.active: List[int] = []
        self.prefill = False
        self._layers = {}           # layer number -> the cache's layer
        self._slots = None          # the active slots on the device
        self._groups = None         # (slots, shared) of _prefix
        self._prefix = None

    @classmethod
    def from_config(cls, config, max_slots: int, max_sequence_length: int,
                    page_size: int = 64, num_pages: Optional[int] = None,
                    device="cuda") -> "PagedInferenceContext":
        if getattr(config, "multi_latent_attention", False) or \
                config.context_parallel_size > 1:
            raise ValueError("PagedInferenceContext: neither multi-latent "
                             "attention nor context parallelism")
        tp = parallel_state.get_tensor_model_parallel_world_size()
        pp = parallel_state.get_pipeline_model_parallel_world_size()
        return cls(config.num_layers // pp, config.num_query_groups // tp,
                   config.kv_channels, max_slots, max_sequence_length,
                   page_size, num_pages, config.params_dtype, device)

    # ------------------------------------------------------------- slots
    def free_slot(self) -> Optional[int]:
        for s in range(self.max_slots):
            if self.host_lengths[s] == 0:
                return s
        return None

    def release(self, slot: int):
        self.cache.free([slot])
        self.host_lengths[slot] = 0
        # the slot's next sequence may share other pages with its neighbours
        self._groups = None

    def fork(self, src: int, dst: List[int]):
        """The slots dst continue what src holds."""
        self.cache.fork([src] * len(dst), dst)
        for t in dst:
            self.host_lengths[t] = self.host_lengths[src]
        self._groups = None

    def reorder_batch(self, indices: torch.Tensor):
        """Row i of the active batch continues row indices[i] (a step of beam
        search)."""
        order = indices.tolist()
        if not all(0 <= i < len(self.active) for i in order):
            raise ValueError(f"PagedInferenceContext: rows {order} of "
                             f"{len(self.active)}")
        self.cache.fork([self.active[i] for i in order], self.active)
        lengths = [self.host_lengths[self.active[i]] for i in order]
        for s, n in zip(self.active, lengths):
            self.host_lengths[s] = n
        self._groups = None

    def _check(self, slots: List[int], more: List[int], empty: bool):
        """What the host can see to be wrong of tokens to come."""
        if len(more) != len(slots) or len(set(slots)) < len(slots) or \
                not all(0 <= s < self.max_slots for s in slots):
            raise ValueError(f"PagedInferenceContext: slots {slots} of "
                             f"{self.max_slots}, each once, with a number of "
                             f"tokens each, got {len(more)}")
        used = [s for s in slots if empty and self.host_lengths[s]]
        if used:
            raise ValueError(f"PagedInferenceContext: slots in use: {used}; "
                             "release() empties them")
        full = [s for s, n in zip(slots, more)
                if self.host_lengths[s] + n > self.max_sequence_length]
        if full:
            raise ValueError(f"PagedInferenceContext: slots {full} would "
                             "hold more than max_sequence_length "
                             f"{self.max_sequence_length}")

    def _set_slots(self, slots: List[int]):
        if self._slots is None or slots != self.active:
            self._slots = torch.tensor(slots, dtype=torch.int32,
                                       device=self.cache.pages.device)
        self.active = list(slots)

    def begin_prompts(self, slots: List[int], lengths: List[int]):
        """The next call of the model is one stream of these prompts, in
        slots that hold nothing."""
        self._check(slots, lengths, True)
        self._set_slots(slots)
        self.prefill = True
        self.cache.extend(self._slots, lengths)
        cu = [0]
        for n in lengths:
            cu.append(cu[-1] + n)
        cu = torch.tensor(cu, dtype=torch.int32,
                          device=self.cache.pages.device)
        self._packing = PackedSeqParams(cu_seqlens_q=cu, cu_seqlens_kv=cu,
                                        max_seqlen_q=max(lengths),
                                        max_seqlen_kv=max(lengths))
        self._positions = torch.cat([
            torch.arange(n, device=self.cache.pages.device)
            for n in lengths])
        for s, n in zip(slots, lengths):
            self.host_lengths[s] = n

    def set_active(self, slots: List[int], prefill: bool = False,
                   shared: Optional[List[Tuple[int, int]]] = None):
        """The next call of the model is one token for each of the slots;
        ``shared`` says how the batch begins, as (rows, tokens) of groups of
        rows that share as many first tokens."""
        assert not prefill, "begin_prompts() admits prompts"
        self._check(slots, [1] * len(slots), False)
        self._set_slots(slots)
        self.prefill = False
        self.cache.extend(self._slots, 1)
        # where no page was left an empty slot stays so, which check() reports;
        # its row still indexes tables of positions
        self._positions = (self.cache.lengths[self._slots.long()].long()
                           - 1).clamp_(min=0)
        key = (tuple(slots), tuple(shared or ()))
        if self._groups != key:
            self._groups = key
            self._prefix = self._shared_prefix(shared or [])

    def _shared_prefix(self, shared) -> Optional[SharedPrefix]:
        if not any(rows > 1 and n for rows, n in shared):
            return None
        ends = [0]
        for rows, _ in shared:
            ends.append(ends[-1] + rows)
        lengths = [n if rows > 1 else 0 for rows, n in shared]
        ints = dict(dtype=torch.int32, device=self.cache.pages.device)
        return SharedPrefix(
            rows=torch.tensor(ends, **ints),
            lengths=torch.tensor(lengths, **ints),
            max_rows=max(r for (r, _), n in zip(shared, lengths) if n),
            max_length=max(lengths))

    def advance(self, n: int):
        for s in self.active:
            self.host_lengths[s] += n

    # ------------------------------------------------------- for the layers
    def update_kv_cache(self, layer_number, key, value):
        raise NotImplementedError(
            "a paged cache is read through attend(): this layer's attention "
            "does not know it")

    def row_positions(self) -> torch.Tensor:
        """Each new token's place in its sequence."""
        return self._positions

    def attend(self, layer_number: int, query: torch.Tensor,
               key: torch.Tensor, value: torch.Tensor,
               softmax_scale: Optional[float] = None) -> torch.Tensor:
        """query [tokens, 1, heads, hd] of packed prompts, or [1, rows, heads,
        hd] of a decode step, with its new key and value: they go to the
        cache, and the query attends over its sequence."""
        layer = self._layers.setdefault(layer_number, len(self._layers))
        cache = self.cache
        if self.prefill:
            cache.write(layer, key[:, 0], value[:, 0], self._slots,
                        self._packing.cu_seqlens_q)
            out = packed_attention(query, key, value, self._packing,
                                   softmax_scale=softmax_scale)
        else:
            cache.write(layer, key[0], value[0], self._slots)
            out = paged_attention(
                query[0], cache.keys(layer), cache.values(layer),
                cache.page_tables, cache.lengths, slots=self._slots,
                shared_prefix=self._prefix, softmax_scale=softmax_scale,
                max_length=max(self.host_lengths[s]
                               for s in self.active) + 1).unsqueeze(0)
        return out.reshape(out.shape[0], out.shape[1], -1)

    def attention_weights(self, layer_number: int, query: torch.Tensor,
                          key: torch.Tensor,
                          softmax_scale: float) -> torch.Tensor:
        """For tracers, after attend() of the same tensors: what it weighed
        the values with, in 32 bits.  [1, heads, tokens, tokens] of packed
        prompts, [rows, heads, 1, longest] of a decode step."""
        heads, d = query.shape[2:]
        groups = key.shape[2]
        if self.prefill:
            t = query.shape[0]
            q = query.permute(1, 2, 0, 3).float().reshape(groups, -1, d)
            k = key.permute(1, 2, 3, 0).float()[0]          # [groups, d, t]
            hide = packed_attention_mask(self._packing.cu_seqlens_q, t)
            shape = (1, heads, t, t)
        else:
            longest = max(self.host_lengths[s] for s in self.active) + 1
            cache, rows = self.cache, self._slots.long()
            pages = cache.page_tables[rows, :-(-longest // cache.page_size)]
            k = cache.keys(self._layers[layer_number])[
                pages.clamp(min=0).long()]      # [rows, pages, groups, page, d]
            k = k.permute(0, 2, 4, 1, 3).flatten(3)[..., :longest].float()
            q = query[0].float().view(len(rows), groups, -1, d)
            hide = torch.arange(longest, device=k.device) >= \
                cache.lengths[rows, None]
            hide = hide[:, None, None]
            shape = (len(rows), heads, 1, longest)
        scores = torch.matmul(q, k).view(shape) * softmax_scale
        return torch.softmax(scores.masked_fill(hide, float("-inf")), -1)
