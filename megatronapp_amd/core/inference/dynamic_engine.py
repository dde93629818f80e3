"""Continuous-batching inference engine (reference
core/inference/engines/dynamic_engine.py:182).

Requests join and leave the decode batch independently: a waiting
request is admitted by prefilling its prompt into a free KV slot; every
``step()`` then runs ONE decode forward for all running slots (per-row
positions + padding masks via DynamicInferenceContext), samples, and
retires finished rows.  ``generate`` drives steps until a set of
prompts drains, but ``add_request``/``step`` are the real API —
requests can be added while others are mid-generation.

With ``kv_page_size`` the cache is paged (PagedInferenceContext): waiting
prompts that fit are prefilled as one packed stream, a decode step reads the
pages where they lie, and ``add_parallel_requests`` continues one prompt
several times over pages that are shared.  A request is admitted when the
pages that it may come to need are left.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional

import torch

from .sampling_params import SamplingParams
from .dynamic_context import DynamicInferenceContext
from .paged_context import PagedInferenceContext
from .static_engine import InferenceRequest
from .text_generation_controller import TextGenerationController
from .. import parallel_state
from ..tensor_parallel.mappings import gather_from_tensor_model_parallel_region


@dataclass
class _Running:
    request_id: int
    prompt: str
    prompt_tokens: List[int]
    sampling: SamplingParams
    slot: int
    generated: List[int] = field(default_factory=list)
    pending_token: Optional[int] = None   # sampled, not yet decoded
    family: int = -1                      # requests of one prompt


@dataclass
class _Family:
    """Requests that continue one prompt, and the pages set aside for them:
    those that all share, and the most that each may need beside them."""
    members: int
    shared_tokens: int
    shared_pages: int
    own_pages: int


class DynamicInferenceEngine:
    def __init__(self, controller: TextGenerationController,
                 max_batch_size: int = 8,
                 max_sequence_length: int = 2048,
                 kv_page_size: Optional[int] = None,
                 kv_num_pages: Optional[int] = None):
        self.controller = controller
        self.max_sequence_length = max_sequence_length
        self.paged = kv_page_size is not None
        self._families: Dict[int, _Family] = {}
        self.waiting: List[_Running] = []
        self.running: List[_Running] = []
        self.finished: Dict[int, InferenceRequest] = {}
        self._next_id = 0
        self._device = ("cuda" if torch.cuda.is_available() else "cpu")
        if self.paged:
            self.context = PagedInferenceContext.from_config(
                controller.model.config, max_batch_size, max_sequence_length,
                kv_page_size, kv_num_pages, self._device)
            self._pages_left = self.context.cache.num_pages
        else:
            self.context = DynamicInferenceContext(max_batch_size,
                                                   max_sequence_length)

    # ------------------------------------------------------------- intake
    def add_request(self, prompt: str,
                    sampling: Optional[SamplingParams] = None) -> int:
        return self.add_parallel_requests(prompt, sampling, 1)[0]

    def add_parallel_requests(self, prompt: str,
                              sampling: Optional[SamplingParams] = None,
                              num_samples: int = 1) -> List[int]:
        """One prompt, continued ``num_samples`` times; the requests' ids.
        With a paged cache the prompt is prefilled once and its pages are
        shared."""
        sampling = sampling or SamplingParams()
        if num_samples < 1:
            raise ValueError("num_samples must be positive")
        toks = self.controller.tokenize_prompts([prompt])[0]
        ids = list(range(self._next_id, self._next_id + num_samples))
        if self.paged:
            self._families[ids[0]] = self._family_of(toks, sampling,
                                                     num_samples)
        self._next_id += num_samples
        self.waiting += [_Running(rid, prompt, toks, sampling, slot=-1,
                                  family=ids[0]) for rid in ids]
        return ids

    def _family_of(self, toks, sampling, members) -> _Family:
        if not toks:
            raise ValueError("a prompt without tokens")
        # the last token that is generated never gets to the cache
        longest = len(toks) + max(sampling.num_tokens_to_generate, 1) - 1
        if longest > self.max_sequence_length:
            raise ValueError(
                f"{len(toks)} prompt tokens and "
                f"{sampling.num_tokens_to_generate} to generate are more "
                f"than max_sequence_length {self.max_sequence_length}")
        page = self.context.cache.page_size
        shared = len(toks) // page
        family = _Family(members, shared * page, shared,
                         -(-longest // page) - shared)
        if members > self.context.max_slots or \
                shared + members * family.own_pages > \
                self.context.cache.num_pages:
            raise ValueError(
                f"{members} request(s) of {longest} tokens do not fit into "
                f"the cache at once")
        return family

    def has_unfinished_requests(self) -> bool:
        return bool(self.waiting or self.running)

    # -------------------------------------------------------------- logic
    def _logits_last(self, logits):
        last = logits[:, -1, :]
        if parallel_state.get_tensor_model_parallel_world_size() > 1:
            last = gather_from_tensor_model_parallel_region(last)
        return last

    def _admit_paged(self):
        """Prefills the waiting families that slots and pages are left for,
        in order, as one packed stream; the members of each fork from its
        first one."""
        ctx = self.context
        slots = [s for s in range(ctx.max_slots) if ctx.host_lengths[s] == 0]
        batch: List[List[_Running]] = []
        tokens = 0
        while self.waiting:
            family = self._families[self.waiting[0].family]
            pages = family.shared_pages + family.members * family.own_pages
            tokens += len(self.waiting[0].prompt_tokens)
            if family.members > len(slots) or pages > self._pages_left:
                break
            # the stream has logits for all its tokens: no more of them than
            # one prompt may have, the others go with the next step
            if batch and tokens > self.max_sequence_length:
                break
            members = self.waiting[:family.members]
            del self.waiting[:family.members]
            for req in members:
                req.slot = slots.pop(0)
            self._pages_left -= pages
            batch.append(members)
        if not batch:
            return
        prompts = [members[0].prompt_tokens for members in batch]
        ctx.begin_prompts([members[0].slot for members in batch],
                          [len(p) for p in prompts])
        toks = torch.tensor([[t for p in prompts for t in p]],
                            dtype=torch.long, device=self._device)
        with torch.no_grad():
            logits = self.controller.model(
                toks, ctx.row_positions().unsqueeze(0), inference_context=ctx)
        end = 0
        for members, prompt in zip(batch, prompts):
            end += len(prompt)
            if len(members) > 1:
                ctx.fork(members[0].slot, [r.slot for r in members[1:]])
            new = self.controller.sample(
                self._logits_last(logits[:, :end]).expand(len(members), -1),
                members[0].sampling)
            for req, tok in zip(members, new.tolist()):
                req.pending_token = tok
                self.running.append(req)

    def _shared(self):
        """How the running rows share pages: (rows, tokens) of each family;
        members stand next to each other."""
        groups, last = [], None
        for req in self.running:
            if req.family == last:
                groups[-1][0] += 1
            else:
                groups.append([1, self._families[req.family].shared_tokens])
                last = req.family
        return [tuple(g) for g in groups]

    def _release_pages(self, req: _Running):
        family = self._families[req.family]
        family.members -= 1
        self._pages_left += family.own_pages
        if family.members == 0:
            self._pages_left += family.shared_pages
            del self._families[req.family]

    def _admit(self):
        if self.paged:
            self._admit_paged()
            return
        ctx = self.context
        while self.waiting:
            slot = ctx.free_slot()
            if slot is None:
                return
            req = self.waiting.pop(0)
            req.slot = slot
            plen = len(req.prompt_tokens)
            ctx.set_active([slot], prefill=True)
            toks = torch.tensor([req.prompt_tokens], dtype=torch.long,
                                device=self._device)
            pos = torch.arange(plen, device=self._device).unsqueeze(0)
            with torch.no_grad():
                logits = self.controller.model(toks, pos,
                                               inference_context=ctx)
            ctx.advance(plen)
            tok = int(self.controller.sample(
                self._logits_last(logits), req.sampling))
            req.pending_token = tok
            self.running.append(req)

    def _retire(self, req: _Running, include_pending: bool):
        if include_pending and req.pending_token is not None:
            req.generated.append(req.pending_token)
        self.context.release(req.slot)
        if self.paged:
            self._release_pages(req)
            self.context.cache.check()
        gen = torch.tensor(req.generated, dtype=torch.long)
        out = InferenceRequest(
            prompt=req.prompt, prompt_tokens=req.prompt_tokens,
            generated_tokens=gen, generated_log_probs=None)
        out.generated_text = self.controller.detokenize(gen)
        out.request_id = req.request_id
        self.finished[req.request_id] = out

    def step(self):
        """Admit waiting requests, run one decode step, retire rows."""
        self._admit()
        if not self.running:
            return
        # retire rows whose pending token ends them BEFORE decoding it
        still = []
        for req in self.running:
            t = req.pending_token
            ends = (t is not None and
                    ((req.sampling.termination_id >= 0 and
                      t == req.sampling.termination_id) or
                     len(req.generated) + 1 >=
                     req.sampling.num_tokens_to_generate))
            if ends:
                self._retire(req, include_pending=True)
            else:
                still.append(req)
        self.running = still
        if not self.running:
            return

        ctx = self.context
        slots = [r.slot for r in self.running]
        if self.paged:
            ctx.set_active(slots, shared=self._shared())
        else:
            ctx.set_active(slots, prefill=False)
        toks = torch.tensor([[r.pending_token] for r in self.running],
                            dtype=torch.long, device=self._device)
        pos = ctx.row_positions().unsqueeze(1)
        with torch.no_grad():
            logits = self.controller.model(toks, pos, inference_context=ctx)
        ctx.advance(1)
        new = self.controller.sample(self._logits_last(logits),
                                     self.running[0].sampling)
        for i, req in enumerate(self.running):
            req.generated.append(req.pending_token)
            req.pending_token = int(new[i])

    # ---------------------------------------------------------- frontend
    @torch.no_grad()
    def generate(self, prompts: List[str],
                 sampling_params: Optional[SamplingParams] = None
                 ) -> List[InferenceRequest]:
        ids = [self.add_request(p, sampling_params) for p in prompts]
        while self.has_unfinished_requests():
            self.step()
        return [self.finished[i] for i in ids]


def get_dynamic_inference_engine(model, tokenizer, max_batch_size=8,
                                 max_sequence_length=2048, kv_page_size=None,
                                 kv_num_pages=None):
    return DynamicInferenceEngine(
        TextGenerationController(model, tokenizer, use_hip_graphs=False),
        max_batch_size, max_sequence_length, kv_page_size, kv_num_pages)
