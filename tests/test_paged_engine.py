"""The dynamic engine over a paged cache: prompts in one packed stream, pages
shared by the samples of a prompt, and the same tokens as without pages."""

import pytest
import torch

from megatronapp_amd.core.inference.dynamic_engine import (
    get_dynamic_inference_engine)
from megatronapp_amd.core.inference.sampling_params import SamplingParams
from megatronapp_amd.core.models.gpt import GPTModel
from megatronapp_amd.core.models.gpt.gpt_layer_specs import (
    get_gpt_layer_local_spec)
from megatronapp_amd.core.tensor_parallel.random import (
    model_parallel_cuda_manual_seed)
from megatronapp_amd.core.transformer_config import TransformerConfig
from megatronapp_amd.training.tokenizer import NullTokenizer
from tests.utils import destroy, initialize_model_parallel

gpu = pytest.mark.gpu

PROMPTS = ["5 9 13", "2 4 6 8 10 12", "7", "1 3 5 7 9",
           " ".join(str(i % 120) for i in range(40))]


def _model(position="rope", device="cpu", groups=None, hidden=64, heads=4,
           use_flash=True, **kw):
    initialize_model_parallel()
    model_parallel_cuda_manual_seed(9)
    torch.manual_seed(9)
    cfg = TransformerConfig(
        num_layers=2, hidden_size=hidden, num_attention_heads=heads,
        num_query_groups=groups, ffn_hidden_size=128, hidden_dropout=0.0,
        attention_dropout=0.0, position_embedding_type=position, **kw)
    with torch.device(device):
        model = GPTModel(
            config=cfg,
            transformer_layer_spec=get_gpt_layer_local_spec(
                use_flash=use_flash),
            vocab_size=128, max_sequence_length=128,
            position_embedding_type=position)
    return model.eval()


def _engine(model, slots=3, pages=None, page=16):
    return get_dynamic_inference_engine(
        model, NullTokenizer(127), max_batch_size=slots,
        max_sequence_length=64, kv_page_size=page, kv_num_pages=pages)


def _cpu_only():
    if torch.cuda.is_available():
        pytest.skip("the engine's model runs on the GPU here")


@pytest.mark.parametrize("position,groups,use_flash", [
    ("rope", None, True), ("rope", 2, False), ("learned_absolute", 1, True)])
def test_same_tokens_as_without_pages(position, groups, use_flash):
    _cpu_only()
    model = _model(position, groups=groups, use_flash=use_flash)
    sp = SamplingParams(num_tokens_to_generate=20, top_k=1)
    want = get_dynamic_inference_engine(
        model, NullTokenizer(127), max_batch_size=3, max_sequence_length=64)
    paged = _engine(model)
    for e in (want, paged):       # two now, the others after two steps
        ids = [e.add_request(p, sp) for p in PROMPTS[:2]]
        e.step()
        e.step()
        ids += [e.add_request(p, sp) for p in PROMPTS[2:]]
        while e.has_unfinished_requests():
            e.step()
        e.texts = [e.finished[i].generated_text for i in ids]
    assert paged.texts == want.texts
    cache = paged.context.cache
    assert cache.free_pages() == cache.num_pages == paged._pages_left
    destroy()


def test_places_not_written_do_not_matter_without_pages():
    """The window of a batch covers places that its shorter rows have not
    written: the cache's memory must not hold NaN there."""
    from megatronapp_amd.core.inference.dynamic_context import (
        DynamicInferenceContext)
    dirty = [torch.full((64 * 2 * 2 * 8,), float("nan")) for _ in range(8)]
    del dirty
    ctx = DynamicInferenceContext(2, 64)
    kv = torch.randn(5, 1, 2, 8)
    ctx.set_active([1], prefill=True)
    ctx.update_kv_cache(0, kv, kv)
    for x in ctx.key_value_memory_dict[0]:
        assert torch.isfinite(x).all()


def test_samples_share_their_prompt():
    _cpu_only()
    model = _model()
    sp = SamplingParams(num_tokens_to_generate=20, top_k=1)
    alone = _engine(model).generate([PROMPTS[4]], sp)[0].generated_text
    e = _engine(model, slots=4)
    ids = e.add_parallel_requests(PROMPTS[4], sp, 3)
    other = e.add_request(PROMPTS[0], sp)
    e.step()
    # two full pages of the prompt's 40 tokens, held by all three
    tables = e.context.cache.page_tables
    slots = [r.slot for r in e.running[:3]]
    assert len({tuple(tables[s, :2].tolist()) for s in slots}) == 1
    assert len({int(tables[s, 2]) for s in slots}) == 3
    assert e.context._prefix.rows.tolist() == [0, 3, 4]
    assert e.context._prefix.lengths.tolist() == [32, 0]
    while e.has_unfinished_requests():
        e.step()
    assert [e.finished[i].generated_text for i in ids] == [alone] * 3
    assert e.finished[other].generated_text == \
        _engine(model).generate([PROMPTS[0]], sp)[0].generated_text
    assert e.context.cache.free_pages() == e.context.cache.num_pages
    # samples that part ways
    torch.manual_seed(0)
    ids = e.add_parallel_requests(
        PROMPTS[4], SamplingParams(num_tokens_to_generate=10,
                                   temperature=5.0), 3)
    while e.has_unfinished_requests():
        e.step()
    assert len({e.finished[i].generated_text for i in ids}) == 3
    destroy()


def test_without_pages_samples_are_separate_requests():
    _cpu_only()
    model = _model()
    sp = SamplingParams(num_tokens_to_generate=4, top_k=1)
    e = get_dynamic_inference_engine(model, NullTokenizer(127),
                                     max_batch_size=2, max_sequence_length=64)
    ids = e.add_parallel_requests(PROMPTS[1], sp, 3)
    while e.has_unfinished_requests():
        e.step()
    assert len({e.finished[i].generated_text for i in ids}) == 1
    destroy()


def test_requests_wait_for_pages():
    _cpu_only()
    model = _model()
    sp = SamplingParams(num_tokens_to_generate=20, top_k=1)
    want = [_engine(model).generate([p], sp)[0].generated_text
            for p in PROMPTS]
    e = _engine(model, slots=5, pages=5)     # at most two at a time
    got = [r.generated_text for r in e.generate(PROMPTS, sp)]
    assert got == want
    assert e.context.cache.free_pages() == 5 == e._pages_left
    for prompt, n, kw in ((PROMPTS[4], 2, {}), (PROMPTS[0], 6, {}),
                          (PROMPTS[0], 0, {}), ("", 1, {}),
                          (PROMPTS[4], 1, dict(num_tokens_to_generate=26))):
        with pytest.raises(ValueError):
            e.add_parallel_requests(
                prompt, SamplingParams(**{"num_tokens_to_generate": 20, **kw}),
                n)
    assert not e.has_unfinished_requests()
    destroy()


def test_a_step_admits_no_more_than_one_longest_prompt():
    _cpu_only()
    model = _model()
    sp = SamplingParams(num_tokens_to_generate=3, top_k=1)
    want = _engine(model).generate([PROMPTS[4]], sp)[0].generated_text
    e = _engine(model, slots=4)
    seen, inner = [], e.context.begin_prompts
    e.context.begin_prompts = lambda s, n: seen.append(n) or inner(s, n)
    out = e.generate([PROMPTS[4]] * 3 + [PROMPTS[0]], sp)   # 40 of 64 each
    assert seen == [[40], [40], [40, 3]]
    assert [r.generated_text for r in out[:3]] == [want] * 3
    destroy()


def test_beams_reorder_by_fork():
    _cpu_only()
    model = _model()
    ctx = _engine(model, slots=3).context
    toks = torch.tensor([[5, 9, 13, 2] * 5 + [1, 2]])
    with torch.no_grad():
        ctx.begin_prompts([0], [22])
        model(toks, ctx.row_positions().unsqueeze(0), inference_context=ctx)
        ctx.fork(0, [1, 2])

        def step(words):
            ctx.set_active([0, 1, 2])
            out = model(torch.tensor([[w] for w in words]),
                        ctx.row_positions().unsqueeze(1),
                        inference_context=ctx)
            ctx.advance(1)
            return out[:, -1]

        first = step([3, 4, 5])
        ctx.reorder_batch(torch.tensor([2, 0, 2]))
        second = step([6, 7, 8])
        ctx.cache.check()
        # what each beam now holds, from the beginning
        for i, words in enumerate([[5, 6], [3, 7], [5, 8]]):
            whole = torch.cat([toks, torch.tensor([words])], 1)
            want = model(whole, torch.arange(24).unsqueeze(0))
            assert torch.allclose(second[i], want[0, -1], atol=1e-4)
    assert first.shape == second.shape
    destroy()


def test_refused_contexts():
    from megatronapp_amd.core.inference.paged_context import (
        PagedInferenceContext)
    with pytest.raises(ValueError, match="head size"):
        PagedInferenceContext(1, 1, 96, 1, 64, device="cuda")
    with pytest.raises(ValueError, match="16 bit|bf16"):
        PagedInferenceContext(1, 1, 64, 1, 64, dtype=torch.float32,
                              device="cuda")


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_generation_on_the_gpu(dtype):
    """Prompts of unlike lengths, samples of one prompt and forks, on the
    kernels.  The step's logits are those of the whole sequence run at once:
    a 2-layer model of order-one activations; every rounding is off by at
    most h relative, some 20 of them follow one another in each layer (QKV,
    rope, P, the attention's output, projection, residuals, norms, MLP) and
    those of the two runs are separate, so 2 * 2 * 20 h of the largest logit
    bound the difference."""
    model = _model(device="cuda", hidden=256, heads=4, groups=2,
                   **{dtype: True})
    e = _engine(model, slots=6)
    sp = SamplingParams(num_tokens_to_generate=12, top_k=1)
    seen = []
    inner = e._logits_last
    e._logits_last = lambda x: seen.append(inner(x)) or seen[-1]
    ids = e.add_parallel_requests(PROMPTS[4], sp, 3)
    ids += [e.add_request(p, sp) for p in PROMPTS[:3]]
    order = []
    while e.has_unfinished_requests():
        e.step()
        order.append([r.request_id for r in e.running])
    h = torch.finfo(getattr(torch, "bfloat16" if dtype == "bf16"
                            else "float16")).eps / 2
    steps = [x for x in seen if x.shape[0] == 6][:11]
    assert len(steps) == 11
    for row, rid in enumerate(order[0]):
        r = e.finished[rid]
        whole = r.prompt_tokens + r.generated_tokens.tolist()
        n = len(r.prompt_tokens)
        with torch.no_grad():
            want = model(torch.tensor([whole], device="cuda"),
                         torch.arange(len(whole), device="cuda")[None])[0]
        for t, x in enumerate(steps):
            off = (x[row].float() - want[n + t].float()).abs().max()
            assert off <= 80 * h * want[n + t].float().abs().max(), (rid, t)
    texts = [e.finished[i].generated_text for i in ids[:3]]
    assert texts[0] == texts[1] == texts[2]
    assert e.context.cache.free_pages() == e.context.cache.num_pages
    destroy()


@gpu
def test_all_of_them_as_a_server_would():
    """Prompts packed, written, forked, extended, compacted and attended over
    with shared pages, against attention over each whole sequence."""
    from megatronapp_amd.core.inference import (PagedKVCache, SharedPrefix,
                                                paged_attention)
    from megatronapp_amd.core.packed_seq_params import PackedSeqParams
    from megatronapp_amd.core.transformer.packed_attention import (
        packed_attention)
    nh, ng, d, dev = 8, 2, 64, "cuda"
    gen = torch.Generator().manual_seed(2)

    def randn(*shape):
        return torch.randn(*shape, generator=gen).bfloat16().to(dev)

    cache = PagedKVCache(2, 64, 16, ng, d, 8, 256)
    lens = [70, 33, 5]
    cu = torch.tensor([0, 70, 103, 108], dtype=torch.int32, device=dev)
    kv = randn(2, 2, 108, ng, d)
    cache.extend([0, 1, 2], lens)
    for layer in range(2):
        cache.write(layer, kv[layer, 0], kv[layer, 1], [0, 1, 2], cu)
    held = {s: kv[:, :, a:b] for s, (a, b) in enumerate(
        zip([0, 70, 103], [70, 103, 108]))}
    q = randn(108, nh, d)
    prompt = packed_attention(q, kv[0, 0], kv[0, 1],
                              PackedSeqParams(cu_seqlens_q=cu))
    cache.free([2])
    cache.fork([0, 0, 1], [3, 4, 2])
    held.update({3: held[0], 4: held[0], 2: held[1]})
    for turn in range(20):
        slots = [0, 3, 4, 1, 2]
        new = randn(2, 2, 5, ng, d)
        cache.extend(slots, 1)
        for layer in range(2):
            cache.write(layer, new[layer, 0], new[layer, 1], slots)
        for i, s in enumerate(slots):
            held[s] = torch.cat([held[s], new[:, :, i:i + 1]], 2)
        if turn == 10:
            cache.compact()
    cache.check()
    s = torch.tensor(slots, dtype=torch.int32, device=dev)
    prefix = SharedPrefix(
        rows=torch.tensor([0, 3, 5], dtype=torch.int32, device=dev),
        lengths=torch.tensor([64, 32], dtype=torch.int32, device=dev),
        max_rows=3, max_length=64)
    q1 = randn(5, nh, d)
    got = paged_attention(q1, cache.keys(1), cache.values(1),
                          cache.page_tables, cache.lengths, slots=s,
                          shared_prefix=prefix)
    h = torch.finfo(torch.bfloat16).eps / 2

    def near(got, q, k, v):      # one query over k, v [n, ng, d]
        for x in range(nh):
            kk, vv = (t[:, x * ng // nh].double() for t in (k, v))
            w = torch.softmax(kk @ q[x].double() / d ** 0.5, 0)
            o = w @ vv
            room = 1.05 * h * (o.abs() + w @ vv.abs())
            assert ((got[x].double() - o).abs() <= room).all()

    for i, slot in enumerate(slots):
        near(got[i], q1[i], held[slot][1, 0], held[slot][1, 1])
    for t in (0, 15, 16, 69, 70, 102, 103, 107):
        a = max(x for x in (0, 70, 103) if x <= t)
        near(prompt[t], q[t], kv[0, 0, a:t + 1], kv[0, 1, a:t + 1])


def _context(slots=3, pages=None, page=16, longest=64, device="cpu"):
    from megatronapp_amd.core.inference.paged_context import (
        PagedInferenceContext)
    return PagedInferenceContext(
        1, 2, 64, slots, longest, page, pages, device=device,
        dtype=torch.float32 if device == "cpu" else torch.bfloat16)


def _new_keys(t, b=1):
    return torch.randn(3, t, b, 2, 64).unbind(0)


def test_a_step_without_pages_left_has_positions_in_range():
    """They index tables of positions, on the GPU without a check."""
    ctx = _context(pages=1)
    ctx.begin_prompts([0], [16])
    ctx.set_active([0, 1])
    assert ctx.row_positions().tolist() == [15, 0]
    with pytest.raises(RuntimeError, match="no free page"):
        ctx.cache.check()


def test_prompts_are_refused_in_slots_in_use():
    """Their tokens would lie behind what the slot holds, and not see it."""
    ctx = _context()
    ctx.begin_prompts([0, 2], [5, 1])
    for slots in ([0], [1, 2]):
        with pytest.raises(ValueError, match="in use"):
            ctx.begin_prompts(slots, [3] * len(slots))
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [5, 0, 1]
    ctx.release(0)
    ctx.begin_prompts([0], [3])
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [3, 0, 1]


def test_sequences_end_at_the_longest():
    """The pages may hold more than that, and tables of positions do not."""
    ctx = _context(longest=20)
    with pytest.raises(ValueError, match="max_sequence_length"):
        ctx.begin_prompts([0, 1], [20, 21])
    ctx.begin_prompts([0, 1], [20, 19])
    ctx.set_active([1])
    ctx.advance(1)
    for slots in ([1], [0], [2, 0]):
        with pytest.raises(ValueError, match="max_sequence_length"):
            ctx.set_active(slots)
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [20, 20, 0]


def test_layers_attention_is_called_and_reports_its_scores():
    """As without pages: hooks on the core attention see each call, and a
    tracer gets the weights, in 32 bits on the CPU within 1e-5 of those."""
    _cpu_only()
    from megatronapp_amd.core.tensor_tracer import (FlagType,
                                                    enable_tensor_tracers)
    model = _model(groups=2)
    tt = enable_tensor_tracers()
    tt.set_num_layers(2)
    tt.tt_flags.set_by_configs({"Raw_attention_score": "True"})
    sp = SamplingParams(num_tokens_to_generate=4, top_k=1)
    calls, seen = [], {}
    for layer in model.decoder.layers:
        layer.self_attention.core_attention.register_forward_hook(
            lambda *a: calls.append(a[0]))
    for paged in (False, True):
        e = _engine(model) if paged else get_dynamic_inference_engine(
            model, NullTokenizer(127), max_batch_size=3,
            max_sequence_length=64)
        seen[paged] = []
        tt.set_report(lambda r: seen[paged].append(r)
                      if r["update_type"] == FlagType.RawAttentionScore.value
                      else None)
        e.generate([PROMPTS[4]], sp)
        assert len(calls) == len(seen[paged]) == 2 * 4   # a prompt, 3 steps
        calls.clear()
        e.generate(PROMPTS[:2], sp)
        calls.clear()
    tt.set_report(None)
    for a, b in zip(seen[False][:8], seen[True][:8]):
        assert a["layer_id"] == b["layer_id"]
        x, y = (torch.tensor(r["result"]).view(r["args"]) for r in (a, b))
        n = min(x.shape[-1], y.shape[-1])
        assert (x[..., :n] - y[..., :n]).abs().max() < 1e-5
        assert (x[..., n:] == 0).all() and (y[..., n:] == 0).all()
    last = seen[True][-1]       # two rows: 3 and 6 tokens, and 3 more
    p = torch.tensor(last["result"]).view(last["args"])
    assert p.shape == (2, 4, 1, 9) and (p[0, ..., 6:] == 0).all()
    assert (p.sum(-1) - 1).abs().max() < 1e-5
    destroy()


@gpu
def test_weights_of_a_decode_step_on_the_gpu():
    """They are the ones that the kernel's output is made with."""
    ctx = _context(device="cuda")
    gen = torch.Generator().manual_seed(6)

    def randn(t, b, heads):
        return torch.randn(t, b, heads, 64, generator=gen).bfloat16().cuda()

    ctx.begin_prompts([0, 2], [20, 33])
    ctx.attend(1, randn(53, 1, 4), randn(53, 1, 2), randn(53, 1, 2))
    ctx.set_active([2, 0])
    q, k, v = randn(1, 2, 4), randn(1, 2, 2), randn(1, 2, 2)
    out = ctx.attend(1, q, k, v, 0.125).view(2, 4, 64).double()
    p = ctx.attention_weights(1, q, k, 0.125).double()
    assert p.shape == (2, 4, 1, 34) and (p[1, ..., 21:] == 0).all()
    table = ctx.cache.page_tables[[2, 0], :3].clamp(min=0).long()
    values = ctx.cache.values(0)[table].permute(0, 2, 1, 3, 4).flatten(
        2, 3)[:, :, :34].double().repeat_interleave(2, 1)
    want = torch.matmul(p, values)[:, :, 0]
    # the weights' rounding before V and the output's own, and 5% for what is
    # in 32 bits
    h = torch.finfo(torch.bfloat16).eps / 2
    room = 1.05 * h * (want.abs() + torch.matmul(p, values.abs())[:, :, 0])
    assert ((out - want).abs() <= room).all()


SURELY = 1 << 20      # a host that expects this much shares pages in any case


@gpu
@pytest.mark.parametrize("page", [16, 64])
def test_shared_pages_after_forks_and_compaction(page):
    """The group's kernel over tables that forks and a compaction left."""
    from megatronapp_amd.core.inference import (PagedKVCache, SharedPrefix,
                                                paged_attention)
    nh, ng, d, dev = 8, 2, 64, "cuda"
    gen = torch.Generator().manual_seed(3)

    def randn(*shape):
        return torch.randn(*shape, generator=gen).bfloat16().to(dev)

    cache = PagedKVCache(1, 64, page, ng, d, 8, 512)
    lens = [200, 3 * page, 9]
    held, slots = {}, [0, 3, 4, 5, 1, 2]
    for s, n in reversed(list(enumerate(lens))):
        kv = randn(2, n, ng, d)
        cache.extend([s], n)
        cache.write(0, kv[0], kv[1], [s],
                    torch.tensor([0, n], dtype=torch.int32, device=dev))
        held[s] = kv
    cache.free([2])
    cache.fork([0, 0, 0, 1], [3, 4, 5, 2])
    held.update({3: held[0], 4: held[0], 5: held[0], 2: held[1]})
    for turn in range(20):
        new = randn(2, len(slots), ng, d)
        cache.extend(slots, 1)
        cache.write(0, new[0], new[1], slots)
        for i, s in enumerate(slots):
            held[s] = torch.cat([held[s], new[:, i:i + 1]], 1)
        if turn == 10:
            cache.compact()
    cache.check()
    ints = dict(dtype=torch.int32, device=dev)
    shared = 200 // page * page
    q = randn(len(slots), nh, d)
    got = paged_attention(
        q, cache.keys(0), cache.values(0), cache.page_tables, cache.lengths,
        slots=torch.tensor(slots, **ints),
        shared_prefix=SharedPrefix(torch.tensor([0, 4, 6], **ints),
                                   torch.tensor([shared, 3 * page], **ints),
                                   4, SURELY))
    h = torch.finfo(torch.bfloat16).eps / 2
    for i, s in enumerate(slots):
        k, v = (x.double().repeat_interleave(nh // ng, 1) for x in held[s])
        w = torch.softmax(torch.einsum("hd,nhd->hn", q[i].double(), k)
                          / d ** 0.5, -1)
        o = torch.einsum("hn,nhd->hd", w, v)
        room = 1.05 * h * (o.abs() + torch.einsum("hn,nhd->hd", w, v.abs()))
        assert ((got[i].double() - o).abs() <= room).all(), s


@gpu
def test_the_engines_steps_share_pages(monkeypatch):
    """A family's steps with the pages that it shares read once: the logits
    of the steps that read them row by row, within the roundings of a model
    of two layers (80 h of the largest, as above)."""
    from megatronapp_amd.core.inference.paged_context import (
        PagedInferenceContext)
    model = _model(device="cuda", hidden=256, heads=4, groups=2, bf16=True)
    sp = SamplingParams(num_tokens_to_generate=8, top_k=1)
    inner = PagedInferenceContext._shared_prefix

    def surely(self, shared):
        prefix = inner(self, shared)
        if prefix is not None:
            prefix.max_length = SURELY
            forced.append(prefix.lengths.tolist())
        return prefix

    seen, forced, texts = {}, [], {}
    for force in (False, True):
        if force:
            monkeypatch.setattr(PagedInferenceContext, "_shared_prefix",
                                surely)
        e = _engine(model, slots=6)
        steps = seen[force] = []
        take = e._logits_last
        e._logits_last = lambda x: steps.append(take(x)) or steps[-1]
        ids = e.add_parallel_requests(PROMPTS[4], sp, 4)
        ids.append(e.add_request(PROMPTS[1], sp))
        while e.has_unfinished_requests():
            e.step()
        texts[force] = [e.finished[i].generated_text for i in ids]
    assert forced and forced[0] == [32, 0]
    h = torch.finfo(torch.bfloat16).eps / 2
    rows = [x for x in seen[False] if x.shape[0] == 5]
    assert len(rows) == 7
    for a, b in zip(rows, [x for x in seen[True] if x.shape[0] == 5]):
        off = (a.float() - b.float()).abs().max()
        assert off <= 80 * h * a.float().abs().max()
        if not torch.equal(a.argmax(-1), b.argmax(-1)):
            break               # from here on they answer different tokens
    assert len(set(texts[True][:4])) == 1
    destroy()


def test_reordering_names_rows_of_the_batch():
    """A number below zero is no row from the end."""
    ctx = _context()
    ctx.begin_prompts([0, 1], [5, 7])
    for order in ([0, -1], [2, 0], [0]):
        with pytest.raises(ValueError):
            ctx.reorder_batch(torch.tensor(order))
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [5, 7, 0]
    ctx.reorder_batch(torch.tensor([1, 0]))
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [7, 5, 0]


def test_calls_name_slots_that_there_are_once():
    ctx = _context()
    ctx.begin_prompts([0, 1], [5, 7])
    for slots in ([2, 2], [3], [-1]):
        with pytest.raises(ValueError, match="slots"):
            ctx.begin_prompts(slots, [4] * len(slots))
    with pytest.raises(ValueError, match="slots"):
        ctx.begin_prompts([2], [4, 4])
    for slots in ([0, 0], [0, 3], [-2]):
        with pytest.raises(ValueError, match="slots"):
            ctx.set_active(slots)
    ctx.cache.check()
    assert ctx.active == [0, 1]
    assert ctx.cache.lengths.tolist() == ctx.host_lengths == [5, 7, 0]
