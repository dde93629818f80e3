"""The paged cache: its state on the GPU against the CPU's in every bit, and
both against what each sequence should hold."""

import random

import pytest
import torch

from megatronapp_amd.core.inference.paged_kv_cache import PagedKVCache

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def make(device="cpu", num_pages=40, page_size=16, slots=6, layers=2,
         groups=2, d=8, longest=200, dtype=torch.bfloat16):
    return PagedKVCache(layers, num_pages, page_size, groups, d, slots,
                        longest, dtype=dtype, device=device)


class Model:
    """What each slot's sequence should hold: a list of token numbers, and
    the values that were written for each."""

    def __init__(self, cache):
        self.cache = cache
        self.tokens = [[] for _ in range(cache.max_slots)]
        self.values = {}
        self.gen = torch.Generator().manual_seed(0)

    def extend(self, slots, counts):
        layers, _, _, groups, _, d = self.cache.pages.shape
        self.cache.extend(slots, counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        kv = torch.randn(layers, 2, cu[-1], groups, d, generator=self.gen).to(
            self.cache.pages)
        index = torch.tensor(cu, dtype=torch.int32, device=kv.device)
        for layer in range(layers):
            self.cache.write(layer, kv[layer, 0], kv[layer, 1], slots, index)
        for s, a, b in zip(slots, cu[:-1], cu[1:]):
            for t in range(a, b):
                name = len(self.values)
                self.values[name] = kv[:, :, t].cpu()
                self.tokens[s].append(name)

    def fork(self, src, dst):
        self.cache.fork(src, dst)
        new = [list(self.tokens[s]) for s in src]
        for t, x in zip(dst, new):
            self.tokens[t] = x

    def free(self, slots):
        self.cache.free(slots)
        for s in slots:
            self.tokens[s] = []

    def check(self):
        c = self.cache
        c.check()
        tables, lengths = c.page_tables.tolist(), c.lengths.tolist()
        refs = [0] * c.num_pages
        for s, want in enumerate(self.tokens):
            assert lengths[s] == len(want)
            used = -(-len(want) // c.page_size)
            assert all(p == -1 for p in tables[s][used:])
            for p in tables[s][:used]:
                refs[p] += 1
            if want:
                ids = torch.tensor(tables[s][:used], device=c.pages.device)
                have = c.pages[:, :, ids].permute(0, 1, 2, 4, 3, 5).flatten(
                    2, 3)[:, :, :len(want)].cpu()
                assert torch.equal(
                    have, torch.stack([self.values[t] for t in want], 2)), s
        assert refs == c.ref_counts.tolist()


def _walk(device, seed, steps=25, **kw):
    rng = random.Random(seed)
    m = Model(make(device, **kw))
    for _ in range(steps):
        slots = rng.sample(range(6), rng.randint(1, 6))
        op = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if op == "extend":
            counts = [rng.choice([0, 1, 1, 3, 16, 31]) for _ in slots]
            counts = [c if len(m.tokens[s]) + c <= 80 else 0
                      for s, c in zip(slots, counts)]
            m.extend(slots, counts)
        elif op == "fork":
            m.fork([rng.randrange(6) for _ in slots], slots)
        elif op == "free":
            m.free(slots[:2])
        else:
            n = int((m.cache.ref_counts > 0).sum())
            m.cache.compact()
            assert int((m.cache.ref_counts[:n] > 0).sum()) == n
        m.check()
    return m.cache


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seed", range(6))
def test_sequences_hold_what_was_written(device, seed):
    _walk(device, seed)


@gpu
@pytest.mark.parametrize("seed", range(4))
def test_gpu_state_is_the_cpus(seed):
    a = _walk("cpu", seed, page_size=32, d=64)
    b = _walk("cuda", seed, page_size=32, d=64)
    for x, y in zip(a.state, b.state):
        assert torch.equal(x, y.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_fork_is_simultaneous(device):
    m = Model(make(device))
    m.extend([0, 1, 2], [20, 33, 16])
    m.fork([1, 0, 0, 2], [0, 1, 2, 3])     # 0 and 1 change places
    m.check()
    # the swap's part-filled pages are new, the full ones are shared
    t = m.cache.page_tables.tolist()
    assert t[1][0] == t[2][0] and t[1][1] != t[2][1]
    m.fork([3], [3])
    m.check()
    m.extend([0, 1, 2, 3], [1, 1, 13, 1])  # after a fork each goes its way
    m.check()
    m.fork([5], [0])                       # of an empty one
    m.check()
    assert m.cache.lengths[0] == 0
    m.free([1, 1])
    m.check()


@pytest.mark.parametrize("device", DEVICES)
def test_what_cannot_be_done_changes_nothing(device):
    m = Model(make(device, num_pages=5))
    m.extend([0, 1], [40, 20])             # 3 + 2 pages
    before = [x.clone() for x in m.cache.state[:4]]

    def refused(message):
        with pytest.raises(RuntimeError, match=message):
            m.cache.check()
        m.cache.check()
        for x, y in zip(before, m.cache.state[:4]):
            assert torch.equal(x, y)

    dev = m.cache.pages.device

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    m.cache.fork([0], [2])
    refused("no free page")
    m.cache.fork(ints(0, 0), ints(2, 2))
    refused("named twice")
    m.cache.fork(ints(0, 9), ints(2, 3))
    refused("out of range")
    m.cache.fork(ints(0), ints(-1))
    refused("out of range")
    m.cache.extend([2], 1)
    refused("no free page")
    m.cache.extend([0], 9999)
    refused("longer")
    m.cache.extend(ints(0, 0), 1)
    refused("twice")
    m.cache.extend(ints(7), 1)
    refused("out of range")
    m.cache.extend([0], ints(-1))
    refused("out of range")
    m.cache.copy_pages(ints(0), ints(77))
    refused("out of the pool")
    m.cache.free(ints(-3, 40))
    refused("out of range")
    x = torch.zeros(1, 2, 8, dtype=torch.bfloat16, device=dev)
    m.cache.write(0, x, x, [3])            # an empty slot
    refused("longer")
    m.cache.lengths[0] = -5
    m.cache.fork([0], [2])
    m.cache.lengths[0] = 40
    refused("longer")
    # a table that was loaded with a page out of the pool
    m.cache.page_tables[0, 2] = 77
    m.cache.fork([0], [2])
    with pytest.raises(RuntimeError, match="out of the pool"):
        m.cache.check()
    m.cache.compact()
    m.cache.free([0])
    m.cache.check()


@pytest.mark.parametrize("device", DEVICES)
def test_compact_and_copy(device):
    m = Model(make(device, num_pages=64, longest=400, slots=9))
    m.extend(list(range(6)), [100, 30, 64, 17, 200, 90])
    m.free([0, 2, 4])
    m.cache.compact()
    m.check()
    live = m.cache.ref_counts > 0
    n = int(live.sum())
    assert bool(live[:n].all()) and m.cache.free_pages() == 64 - n
    before = m.cache.pages.clone()
    m.cache.copy_pages([0, 3], [n, n + 2])
    want = before.clone()
    want[:, :, n], want[:, :, n + 2] = before[:, :, 0], before[:, :, 3]
    assert torch.equal(m.cache.pages, want)
    m.cache.free(list(range(9)))
    m.cache.compact()
    assert m.cache.free_pages() == 64


@pytest.mark.parametrize("device", DEVICES)
def test_many_pages(device):
    """More pages than one sweep of a planning block, more slots than its
    threads."""
    c = make(device, num_pages=9001, slots=1500, layers=1, groups=1, d=8,
             longest=96)
    slots = list(range(1500))
    c.extend(slots, [1 + s % 96 for s in slots])
    c.check()
    tables, at = c.page_tables.tolist(), 0
    for s in slots:                         # lowest first, in order
        used = -(-(1 + s % 96) // 16)
        assert tables[s][:used] == list(range(at, at + used))
        at += used
    c.free(slots[::2])
    c.fork(slots[1:1000:2], slots[0:1000:2])
    c.check()
    assert c.lengths[0] == 2 and c.lengths[999] == 1 + 999 % 96
    held = (c.page_tables >= 0)
    c.compact()
    assert torch.equal(held, c.page_tables >= 0)
    n = int((c.ref_counts > 0).sum())
    assert int(c.page_tables.max()) == n - 1
    want = torch.zeros(9001, dtype=torch.int64)
    ids = c.page_tables[held].long().cpu()
    want.index_add_(0, ids, torch.ones_like(ids))
    assert torch.equal(c.ref_counts.cpu().long(), want)


@pytest.mark.parametrize("device", DEVICES)
def test_load_tables_and_from_state(device):
    m = Model(make(device))
    m.extend([0, 1], [20, 5])
    kept = [x.clone() for x in m.cache.state[1:4]]
    m.cache.free([0])
    m.cache.load_tables(*kept)
    m.check()
    twin = PagedKVCache.from_state(*m.cache.state[:4])
    twin.free([1])
    assert m.cache.lengths[1] == 0          # the same tensors
    with pytest.raises(ValueError, match="lengths"):
        m.cache.load_tables(kept[0], kept[1], kept[2][:2])


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    c = make(device)
    dev = c.pages.device
    for bad in ([0, 0], [6], [-1]):
        with pytest.raises(ValueError):
            c.fork([0] * len(bad), bad)
        with pytest.raises(ValueError):
            c.extend(bad, 1)
    with pytest.raises(ValueError):
        c.fork([0], [1, 2])
    with pytest.raises(ValueError):
        c.free([99])
    with pytest.raises(ValueError):
        c.copy_pages([0, 1], [1, 2])
    with pytest.raises(ValueError):
        c.copy_pages([0], [40])
    with pytest.raises(ValueError):
        c.extend([0], [1, 2])
    with pytest.raises(ValueError):
        c.extend([0], -1)
    with pytest.raises(ValueError):
        c.free(torch.zeros(1, device=dev))
    x = torch.zeros(1, 2, 8, dtype=torch.bfloat16, device=dev)
    for layer, k, v, slots in ((2, x, x, [0]), (0, x.float(), x, [0]),
                               (0, x, x, [0, 1]), (0, x[:, :1], x, [0]),
                               (0, x[0], x[0], [0])):
        with pytest.raises(ValueError):
            c.write(layer, k, v, slots)
    with pytest.raises(ValueError):
        c.write(0, x, x, [0], torch.zeros(3, dtype=torch.int32, device=dev))
    for kw in (dict(page_size=8), dict(page_size=24), dict(num_pages=0),
               dict(d=4)):
        with pytest.raises(ValueError):
            make(device, **kw)
    with pytest.raises(ValueError):
        PagedKVCache.from_state(c.pages, c.ref_counts.long(), c.page_tables,
                                c.lengths)
    with pytest.raises(ValueError):
        PagedKVCache.from_state(c.pages, c.ref_counts[1:], c.page_tables,
                                c.lengths)
    with pytest.raises(ValueError):
        PagedKVCache.from_state(c.pages.transpose(0, 1), c.ref_counts,
                                c.page_tables, c.lengths)


@gpu
def test_views_are_written_from_where_they_lie():
    c = make("cuda", d=64, groups=4)
    fused = torch.randn(3, 4, 192, device="cuda").bfloat16()
    k, v = fused[..., 64:128], fused[..., 128:]
    c.extend([4, 0, 2], 1)
    c.write(1, k, v, [4, 0, 2])
    odd = torch.randn(3, 4, 65, device="cuda").bfloat16()[..., 1:]
    c.write(0, odd, odd, [4, 0, 2])
    c.check()
    for i, s in enumerate([4, 0, 2]):
        p = int(c.page_tables[s, 0])
        assert torch.equal(c.keys(1)[p, :, 0], k[i])
        assert torch.equal(c.values(1)[p, :, 0], v[i])
        assert torch.equal(c.keys(0)[p, :, 0], odd[i])


@gpu
def test_captured_and_replayed_with_forks():
    """Two graphs on one cache: a step of decoding and a reordering of beams;
    replayed in turn they do what eager calls do."""
    def walk(graphed):
        c = make("cuda", num_pages=200, slots=4, d=64)
        slots = torch.arange(4, dtype=torch.int32, device="cuda")
        src = torch.zeros(4, dtype=torch.int32, device="cuda")
        kv = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
        c.extend(slots, [5, 5, 5, 5])

        def step():
            c.extend(slots, 1)
            for layer in range(2):
                c.write(layer, kv[0], kv[1], slots)

        def turn():
            c.fork(src, slots)

        if graphed:
            kept = [x.clone() for x in c.state]
            graphs = []
            for f in (step, turn):
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    f()
                torch.cuda.current_stream().wait_stream(side)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    f()
                graphs.append(g.replay)
            for x, y in zip(c.state, kept):
                x.copy_(y)
            step, turn = graphs
        gen = torch.Generator().manual_seed(3)
        for i in range(40):
            kv.copy_(torch.randn(kv.shape, generator=gen))
            src.copy_(torch.randint(0, 4, (4,), generator=gen))
            step()
            turn()
        torch.cuda.synchronize()
        c.check()
        return c

    a, b = walk(False), walk(True)
    for x, y in zip(a.state, b.state):
        assert torch.equal(x, y)


def test_lengths_that_pass_32_bits_are_refused():
    ints = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="2.31"):
        PagedKVCache.from_state(torch.zeros(1, 2, 1, 1, 512, 8),
                                torch.zeros(1, **ints),
                                torch.zeros(1, 1 << 22, **ints),
                                torch.zeros(1, **ints))
    with pytest.raises(ValueError, match="2.31"):
        PagedKVCache(1, 1, 1 << 20, 1, 8, 1, 1 << 31, device="cpu")


@gpu
def test_contiguous_tokens_off_16_bytes_are_written():
    c = make("cuda", d=64, groups=4)
    odd = torch.randn(3 * 4 * 64 + 1, device="cuda").bfloat16()[1:].view(
        3, 4, 64)
    assert odd.is_contiguous() and odd.data_ptr() % 16 == 2
    c.extend([4, 0, 2], 1)
    c.write(0, odd, odd, [4, 0, 2])
    c.check()
    for i, s in enumerate([4, 0, 2]):
        p = int(c.page_tables[s, 0])
        assert torch.equal(c.keys(0)[p, :, 0], odd[i])
        assert torch.equal(c.values(0)[p, :, 0], odd[i])


@pytest.mark.parametrize("device", DEVICES)
def test_the_cache_holds_values_without_their_derivatives(device):
    from torch.autograd import forward_ad
    c = make(device)
    x = torch.randn(1, 2, 8).to(c.pages).requires_grad_(True)
    c.extend([0], 1)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        c.write(0, dual * 2, dual, [0])
        assert not c.pages.requires_grad
        assert forward_ad.unpack_dual(c.pages).tangent is None
    page = int(c.page_tables[0, 0])
    assert torch.equal(c.keys(0)[page, :, 0], x[0].detach() * 2)
    assert torch.equal(c.values(0)[page, :, 0], x[0].detach())


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_behind_32_bits_are_out_of_range(device):
    c = make(device)
    c.extend([0, 1], [20, 5])
    kept = [x.clone() for x in c.state[:4]]
    far = torch.tensor([1 << 32], device=device)
    zero = torch.tensor([0], device=device)
    x = torch.ones(1, 2, 8, dtype=torch.bfloat16, device=device)
    for call, message in (
            (lambda: c.free(far), "slot out of range"),
            (lambda: c.free(-far), "slot out of range"),
            (lambda: c.fork(far, zero + 1), "slot out of range"),
            (lambda: c.fork(zero, far + 2), "slot out of range"),
            (lambda: c.extend(far, 1), "slot out of range"),
            (lambda: c.extend(zero, far + 1), "longer"),
            (lambda: c.copy_pages(zero, far + 9), "out of the pool"),
            (lambda: c.write(0, x, x, far), "slot out of range"),
            (lambda: c.write(0, x, x, zero, torch.cat([zero, far + 1])),
             "longer")):
        call()
        with pytest.raises(RuntimeError, match=message):
            c.check()
        for a, b in zip(kept, c.state[:4]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_shared_pages_are_not_written_where_an_extension_failed(device):
    """No page is left for the step of a sequence whose last page is full:
    its token must not go there, where the others would read it."""
    m = Model(make(device, num_pages=3))
    m.extend([0], [32])
    m.fork([0], [1])
    m.extend([2], [3])
    before = [x.clone() for x in m.cache.state[:4]]
    x = torch.ones(2, 2, 8, dtype=torch.bfloat16, device=m.cache.pages.device)
    m.cache.extend([1, 2], 1)
    for layer in range(2):
        m.cache.write(layer, x[:1], x[:1], [1])
    with pytest.raises(RuntimeError, match="no free page.*several sequences"):
        m.cache.check()
    for a, b in zip(before, m.cache.state[:4]):
        assert torch.equal(a, b)
    m.free([0])                 # now it is slot 1's alone
    m.cache.write(0, x[:1], x[:1], [1])
    m.cache.check()
    page = int(m.cache.page_tables[1, 1])
    assert (m.cache.keys(0)[page, :, 15] == 1).all()


def test_places_next_to_the_longest_stay_in_32_bits():
    """A kernel's step or piece may end behind the longest sequence."""
    ints = dict(dtype=torch.int32)
    for width, fits in (((1 << 22) - 16, True), ((1 << 22) - 15, False)):
        args = (torch.zeros(1, 2, 1, 1, 512, 8), torch.zeros(1, **ints),
                torch.zeros(1, width, **ints), torch.zeros(1, **ints))
        if fits:
            PagedKVCache.from_state(*args)
        else:
            with pytest.raises(ValueError, match="2.31"):
                PagedKVCache.from_state(*args)
