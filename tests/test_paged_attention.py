"""Attention over paged sequences against the formula in 64 bits.

Tolerances.  With h = eps / 2 of the type: P is rounded before the product
with V and the output at the end, so |o - ref| <= h |ref| + h P|V|; sums,
exponentials and the joining of pieces are in 32 bits, below 1e-5 of the
terms, which 5% on top covers.  fp16 values below its normal range are off by
up to 2^-25."""

import math

import pytest
import torch

from megatronapp_amd.core.inference.paged_attention import (SharedPrefix,
                                                            paged_attention)

gpu = pytest.mark.gpu


def _state(lens, nh=4, ng=2, d=64, page=16, dtype=torch.bfloat16, spare=3,
           device="cuda", seed=0, prefix=0):
    """Rows of these lengths, all with the same `prefix` first tokens, their
    pages in no order."""
    g = torch.Generator().manual_seed(seed)
    shared = prefix // page
    need = [-(-n // page) for n in lens]
    pages = shared + sum(max(0, x - shared) for x in need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    tables, at = [], shared
    width = max(need + [1]) + 1
    for x in need:
        own = max(0, x - shared)
        row = order[:min(shared, x)] + order[at:at + own]
        at += own
        tables.append(row + [-1] * (width - len(row)))

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(device)
    return (randn(len(lens), nh, d) * 2.0, randn(pages, ng, page, d),
            randn(pages, ng, page, d),
            torch.tensor(tables, dtype=torch.int32, device=device),
            torch.tensor(lens, dtype=torch.int32, device=device))


def oracle(q, k, v, tables, lengths, scale=None, slots=None):
    b, nh, d = q.shape
    pages, ng, page = k.shape[:3]
    h = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, nh, d, dtype=torch.float64, device=q.device)
    room = torch.zeros_like(out)
    for i in range(b):
        s = i if slots is None else int(slots[i])
        seen = [(int(tables[s, t // page]), t % page)
                for t in range(int(lengths[s]))]
        seen = [x for x in seen if 0 <= x[0] < pages]
        if not seen:
            continue
        p, t = (torch.tensor(x, device=q.device) for x in zip(*seen))
        kk, vv = k[p, :, t].double(), v[p, :, t].double()   # [n, ng, d]
        for x in range(nh):
            z = kk[:, x * ng // nh] @ q[i, x].double() * scale
            w = torch.softmax(z, 0)
            y = vv[:, x * ng // nh]
            out[i, x] = w @ y
            room[i, x] = h * out[i, x].abs() + (h * w + tiny) @ y.abs() + tiny
    return out, 1.05 * room


def _near(got, want, name=""):
    assert torch.isfinite(got).all(), name
    off = ((got.double() - want[0]).abs() - want[1]).max()
    assert off <= 0, (name, off.item())


def _check(lens, scale=None, **kw):
    s = _state(lens, **kw)
    got = paged_attention(*s, softmax_scale=scale)
    _near(got, oracle(*s, scale=scale), (lens, kw))
    return s, got


# ----------------------------------------------------------------- on the CPU
def test_plain_matches_oracle():
    s = _state([1, 0, 16, 40, 33], dtype=torch.float32, device="cpu", nh=6,
               ng=2, d=8)
    got = paged_attention(*s, softmax_scale=0.4)
    out, _ = oracle(*s, scale=0.4)
    # 32 bits: 41 terms and their exponentials, each off by a few 2^-24
    assert (got.double() - out).abs().max() < 1e-5
    slots = torch.tensor([3, 0, 9, -1], dtype=torch.int32)
    got2 = paged_attention(s[0][:4], *s[1:], slots=slots, softmax_scale=0.4)
    want = oracle(s[0][:2], *s[1:], scale=0.4, slots=[3, 0])[0]
    assert (got2[:2].double() - want).abs().max() < 1e-5
    assert (got2[2:] == 0).all()


def test_plain_leaves_out_pages_out_of_the_pool():
    q, k, v, tables, lengths = _state([40, 40, 16], dtype=torch.float32,
                                      device="cpu", d=8)
    tables[0, 1] = 999
    tables[1, 0] = -7
    tables[2, 0] = k.shape[0]
    got = paged_attention(q, k, v, tables, lengths)
    out, _ = oracle(q, k, v, tables, lengths)
    assert (got.double() - out).abs().max() < 1e-5
    assert (got[2] == 0).all()
    lengths[0] = 100000          # longer than the table
    lengths[1] = -4
    got = paged_attention(q, k, v, tables, lengths)
    assert torch.isfinite(got).all() and (got[1] == 0).all()


def _refused(message, device, **change):
    q, k, v, tables, lengths = _state([20, 20], device=device)
    args = dict(query=q, key_pages=k, value_pages=v, page_tables=tables,
                lengths=lengths)
    args.update({n: f(args) if callable(f) else f for n, f in change.items()})
    with pytest.raises(ValueError, match=message):
        paged_attention(**args)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    def _refuse(message, **change):
        _refused(message, device, **change)

    _refuse("must be", query=lambda a: a["query"][0])
    _refuse("must be", value_pages=lambda a: a["value_pages"][:1])
    _refuse("fit", query=lambda a: a["query"][:, :3])
    _refuse("fit", query=lambda a: a["query"][..., :32])
    _refuse("type", query=lambda a: a["query"].half())
    _refuse("int32", lengths=lambda a: a["lengths"].long())
    _refuse("int32", page_tables=lambda a: a["page_tables"][0])
    _refuse("one length", lengths=lambda a: a["lengths"][:1])
    _refuse("slot", slots=lambda a: a["lengths"][:1])
    _refuse("positive", softmax_scale=0.0)
    _refuse("16", key_pages=lambda a: a["key_pages"][:, :, :8],
            value_pages=lambda a: a["value_pages"][:, :, :8])
    _refuse("longer", shared_prefix=lambda a: SharedPrefix(
        a["lengths"], a["lengths"], 1, 16))
    _refuse("int32", shared_prefix=lambda a: SharedPrefix(
        a["lengths"].long(), a["lengths"][:1], 1, 16))
    _refuse("gradient", query=lambda a: a["query"].requires_grad_(True))


# ----------------------------------------------------------------- on the GPU
@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [
    [1], [0], [15, 16, 17], [31, 32, 33, 0, 1], [127, 128, 129, 500]])
def test_lengths(lens, dtype, d):
    _check(lens, dtype=dtype, d=d)


@gpu
@pytest.mark.parametrize("page", [16, 32, 48, 64, 256])
def test_page_sizes(page):
    _check([1, page - 1, page, page + 1, 5 * page + 3], page=page, d=64)
    _check([700, 2, 300], page=page, d=128, nh=8, ng=1)


@gpu
@pytest.mark.parametrize("nh,ng", [(1, 1), (3, 3), (16, 1), (24, 1), (40, 2),
                                   (32, 8)])
def test_head_layouts(nh, ng):
    _check([70, 3, 190], nh=nh, ng=ng, d=64)
    _check([70, 3, 190], nh=nh, ng=ng, d=128, scale=0.2)


@gpu
@pytest.mark.parametrize("n", [4200, 4300, 4400, 4500])
@pytest.mark.parametrize("d", [64, 128])
def test_any_number_of_pieces(n, d):
    """33 to 36 pieces of one row."""
    _check([n], nh=2, ng=1, d=d)


@gpu
def test_long_rows_and_many_rows():
    _check([9000, 31], nh=4, ng=2, d=128, page=64)
    _check([(i * 37) % 90 for i in range(150)], nh=2, ng=1, d=64)


@gpu
def test_what_lies_behind_the_end_does_not_matter():
    lens = [21, 40, 3]
    s, want = _check(lens, d=64, spare=2)
    k, v = s[1].clone(), s[2].clone()
    used = torch.zeros(k.shape[0], k.shape[2], dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(n):
            used[int(s[3][i, t // 16]), t % 16] = True
    hide = ~used.cuda()[:, None, :, None]
    for x, by in ((k, math.nan), (v, math.inf), (v, math.nan)):
        x.masked_fill_(hide, by)
        assert torch.equal(paged_attention(s[0], k, v, *s[3:]), want)


@gpu
def test_pages_out_of_the_pool_and_lengths_out_of_range():
    q, k, v, tables, lengths = _state([40, 40, 16], d=64)
    tables[0, 1] = 999
    tables[1, 0] = -7
    tables[2, 0] = k.shape[0]
    got = paged_attention(q, k, v, tables, lengths)
    _near(got, oracle(q, k, v, tables, lengths))
    assert (got[2] == 0).all()
    lengths[0] = 1 << 30
    lengths[1] = -4
    got = paged_attention(q, k, v, tables, lengths)
    assert torch.isfinite(got).all() and (got[1] == 0).all()
    slots = torch.tensor([1, 77, -1], dtype=torch.int32, device="cuda")
    assert (paged_attention(q, k, v, tables, lengths, slots=slots)
            == 0).all()


@gpu
def test_slots_strides_and_layouts():
    q, k, v, tables, lengths = _state([21, 200, 33, 0], d=64, nh=4, ng=2)
    slots = torch.tensor([2, 2, 0, 3, 1, 1], dtype=torch.int32,
                         device="cuda")
    wide = torch.randn(6, 2, 4, 3, 64, device="cuda").bfloat16()
    qv = wide[:, 1, :, 1]                      # a view
    got = paged_attention(qv, k, v, tables, lengths, slots=slots)
    want = oracle(qv, k, v, tables, lengths, slots=slots)
    _near(got, want)
    # tokens before heads in a page; a layer of a whole cache
    kt = k.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack([k, v])
    assert torch.equal(paged_attention(qv, kt, both[1], tables, lengths,
                                       slots=slots), got)
    odd = torch.empty(6 * 4 * 64 + 1, device="cuda").bfloat16()[1:].view(
        6, 4, 64)
    odd.copy_(qv)
    assert torch.equal(paged_attention(odd, k, v, tables, lengths,
                                       slots=slots), got)
    # the longest row that the host knows of only cuts the work
    for most in (1, 50, 100000):
        _near(paged_attention(qv, k, v, tables, lengths, slots=slots,
                              max_length=most), want)


@gpu
def test_pages_far_into_a_large_cache():
    """Offsets past 2^31 elements."""
    d, page, ng = 128, 64, 8
    pages = (1 << 31) // (page * ng * d) + 64
    k = torch.zeros(pages, ng, page, d, dtype=torch.bfloat16, device="cuda")
    q, ks, vs, tables, lengths = _state([100, 30], nh=8, ng=ng, d=d,
                                        page=page, spare=0)
    n = ks.shape[0]
    want = paged_attention(q, ks, vs, tables, lengths)
    for name, x in (("k", ks), ("v", vs)):
        k[-n:] = x
        far = torch.where(tables >= 0, tables + pages - n, tables).int()
        if name == "k":
            v = torch.zeros_like(k)
            v[-n:] = vs
    k[-n:] = ks
    assert torch.equal(paged_attention(q, k, v, far, lengths), want)


@gpu
def test_another_stream_and_the_same_bits():
    s, want = _check([900, 17, 260], nh=8, ng=2, d=128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(*s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@gpu
def test_two_captured_graphs():
    """Lengths and queries change between replays; two graphs of one pool
    and eager calls go in turn."""
    s = _state([300, 17, 260], nh=8, ng=2, d=64)
    q, k, v, tables, lengths = s
    graphs, outs = [], []
    for most in (320, 40):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged_attention(*s, max_length=most)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(paged_attention(*s, max_length=most))
        graphs.append(g)
    for i in range(6):
        lengths.copy_(torch.tensor([300 - 40 * i, 17, i * 7],
                                   dtype=torch.int32))
        q.mul_(0.9)
        want = oracle(*s)
        graphs[i % 2].replay()
        _near(outs[i % 2], want)
        graphs[1 - i % 2].replay()
        _near(outs[1 - i % 2], want)
        _near(paged_attention(*s), want)


SURELY = 1 << 20      # a host that expects this much always shares


def _groups(rows, lengths, max_rows=None, max_length=SURELY):
    ends = list(rows)
    return SharedPrefix(
        torch.tensor(ends, dtype=torch.int32, device="cuda"),
        torch.tensor(lengths, dtype=torch.int32, device="cuda"),
        max_rows if max_rows is not None else
        max(b - a for a, b in zip(ends[:-1], ends[1:])),
        max_length)


def _grouped_state(sizes, prefixes, own, **kw):
    """Rows of several groups, each on a prefix of its own."""
    parts, at = [], 0
    for i, (r, p) in enumerate(zip(sizes, prefixes)):
        if r:
            parts.append(_state([p + n for n in own[at:at + r]], prefix=p,
                                seed=i, **kw))
        at += r
    width = max(x[3].shape[1] for x in parts)
    tables, base = [], 0
    for x in parts:
        t = torch.where(x[3] >= 0, x[3] + base, x[3])
        tables.append(torch.nn.functional.pad(t, (0, width - t.shape[1]),
                                              value=-1))
        base += x[1].shape[0]
    return (torch.cat([x[0] for x in parts]), torch.cat([x[1] for x in parts]),
            torch.cat([x[2] for x in parts]), torch.cat(tables).int(),
            torch.cat([x[4] for x in parts]))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_shared_prefix(dtype, d):
    own = [1 + (i * 37) % 90 for i in range(50)]
    s = _grouped_state([50], [640], own, dtype=dtype, d=d, nh=8, ng=2)
    want = oracle(*s)
    for most in (640, 1, SURELY):
        _near(paged_attention(*s, shared_prefix=_groups([0, 50], [640], 50,
                                                        most)), want)
    # a host that knows too few rows
    _near(paged_attention(*s, shared_prefix=_groups([0, 50], [640], 1)),
          want)
    # a part of a page does not count
    _near(paged_attention(*s, shared_prefix=_groups([0, 50], [639])), want)
    # rows outside the group, one of them among them
    _near(paged_attention(*s, shared_prefix=_groups([3, 41], [640])), want)


@gpu
@pytest.mark.parametrize("page", [16, 48, 64])
def test_groups_of_rows(page):
    sizes = [9, 1, 0, 6, 40]
    prefixes = [page * 11, 0, page, page * 30, page * 3]
    own = [(i * 53) % 200 for i in range(sum(sizes))]
    s = _grouped_state(sizes, prefixes, own, page=page, d=64, nh=12, ng=3)
    ends = [0, 9, 10, 10, 16, 56]
    want = oracle(*s)
    for rows in (40, 3):
        _near(paged_attention(*s, shared_prefix=_groups(ends, prefixes,
                                                        rows)), want)
    s2 = _grouped_state(sizes[:2], prefixes[:2], own[:10], page=page, d=128,
                        nh=48, ng=2)
    _near(paged_attention(*s2, shared_prefix=_groups(ends[:3], prefixes[:2])),
          oracle(*s2))


@gpu
def test_a_long_prefix_for_many_rows():
    own = [1 + (i * 37) % 90 for i in range(70)]
    s = _grouped_state([70], [6400], own, d=128, nh=8, ng=2, page=64)
    want = oracle(*s)
    for most in (6400, SURELY):
        _near(paged_attention(*s, shared_prefix=_groups([0, 70], [6400], 70,
                                                        most)), want)


@gpu
def test_groups_with_short_rows_and_bad_pages():
    """Rows shorter than their group's prefix see their own length; bad pages
    of the prefix are left out, whatever the pool's first page holds."""
    own = [5] * 20
    q, k, v, tables, lengths = _grouped_state([20], [320], own, d=64, nh=8)
    lengths[3], lengths[7], lengths[19] = 40, 0, 320
    tables[:, 4] = 9999
    tables[:, 9] = -1
    g = _groups([0, 20], [320])
    want = oracle(q, k, v, tables, lengths)
    got = paged_attention(q, k, v, tables, lengths, shared_prefix=g)
    _near(got, want)
    used = set(tables[:, :21].flatten().tolist())
    if 0 not in used:
        k[0], v[0] = math.nan, math.nan
    else:       # the sequence's own first page: move it to the last
        k, v = torch.cat([k, k[:1]]), torch.cat([v, v[:1]])
        tables[tables == 0] = k.shape[0] - 1
        k[0], v[0] = math.nan, math.nan
    # one more page in the pool: numbers out of it stay out of it
    assert torch.equal(paged_attention(q, k, v, tables, lengths,
                                       shared_prefix=g), got)


@gpu
def test_groups_by_slots_in_a_graph():
    """The groups' rows and lengths, and the rows' slots, change between
    replays."""
    own = [(i * 37) % 60 for i in range(12)]
    s = _grouped_state([4, 8], [160, 64], own, d=64, nh=8, ng=2)
    q, k, v, tables, lengths = s
    slots = torch.arange(12, dtype=torch.int32, device="cuda")
    g = _groups([0, 4, 12], [160, 64])

    def run():
        return paged_attention(q, k, v, tables, lengths, slots=slots,
                               shared_prefix=g, max_length=224)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for ends, shared, order in (
            ([0, 4, 12], [160, 64], range(12)),
            ([0, 4, 12], [32, 16], range(12)),
            ([0, 8, 12], [64, 160], list(range(4, 12)) + list(range(4))),
            ([0, 0, 0], [160, 64], range(12))):
        g.rows.copy_(torch.tensor(ends, dtype=torch.int32))
        g.lengths.copy_(torch.tensor(shared, dtype=torch.int32))
        slots.copy_(torch.tensor(list(order), dtype=torch.int32))
        q.mul_(0.9)
        want = oracle(*s, slots=slots)
        graph.replay()
        _near(out, want)
        graph.replay()
        _near(out, want)
        _near(run(), want)


@gpu
def test_refusals_on_the_gpu():
    q, k, v, tables, lengths = _state([20, 20], d=32)
    with pytest.raises(ValueError, match="head size"):
        paged_attention(q, k, v, tables, lengths)
    q, k, v, tables, lengths = _state([20, 20])
    with pytest.raises(ValueError, match="device"):
        paged_attention(q, k, v, tables.cpu(), lengths)
    with pytest.raises(ValueError, match="head size"):
        paged_attention(q.float(), k.float(), v.float(), tables, lengths)
    assert paged_attention(q[:0], k, v, tables[:1], lengths[:1],
                           slots=lengths[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------ pieces
@gpu
@pytest.mark.parametrize("n", [8200, 8600, 9000, 9200])
def test_many_pieces_of_a_row(n):
    """33 to 36 pieces of 256 keys."""
    _check([n], nh=2, ng=1, d=128)
    _check([n], nh=16, ng=16, d=64)


@gpu
@pytest.mark.parametrize("nh,ng,d", [(32, 32, 64), (40, 8, 128)])
def test_long_rows_among_short_ones(nh, ng, d):
    """A row's length alone gives it further pieces, which lie with other
    rows' ones in blocks that they share."""
    lens = [1 + 7 * i % 90 for i in range(140)]
    for i, n in ((0, 5000), (63, 1025), (64, 2048), (65, 2049), (139, 12345)):
        lens[i] = n
    s = _state(lens, nh=nh, ng=ng, d=d)
    want = oracle(*s)
    for most in (None, 1, 3000):      # only the time depends on it
        _near(paged_attention(*s, max_length=most), want, most)


# ------------------------------------------------------------------- NaN
@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_a_query_of_nan_gives_nan(d):
    """Rows of one piece, of several, and of a group: NaN for the head that
    has it, and what the other heads and rows give stays."""
    own = [1, 40, 300, 3000, 5, 90, 700]
    s = _grouped_state([3, 4], [640, 160], own, d=d, nh=8, ng=2)
    rows = [0, 1, 2, 3, 6]
    q = s[0].clone()
    q[rows, 3] = math.nan
    for kw in ({}, dict(max_length=1),
               dict(shared_prefix=_groups([0, 3, 7], [640, 160]))):
        want = paged_attention(*s, **kw)
        got = paged_attention(q, *s[1:], **kw)
        assert torch.isnan(got[rows, 3]).all(), kw
        got[rows, 3] = want[rows, 3]
        assert torch.equal(got, want), kw


@gpu
def test_keys_of_nan_give_nan():
    """A page whose keys are NaN is a piece, or some waves' part of one,
    without any score."""
    q, k, v, tables, lengths = _state([2000, 100], d=64, page=256)
    k[int(tables[0, 3])] = math.nan
    for most in (None, 1):
        got = paged_attention(q, k, v, tables, lengths, max_length=most)
        assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused(which, device):
    from torch.autograd import forward_ad
    s = list(_state([20, 20], device=device))
    with forward_ad.dual_level():
        s[which] = forward_ad.make_dual(s[which], torch.ones_like(s[which]))
        with torch.no_grad(), pytest.raises(ValueError, match="forward mode"):
            paged_attention(*s)


# ------------------------------------------------------------ sizes of pages
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("page", [528, 1040, 16400])
def test_any_multiple_of_sixteen_is_a_page(page, device):
    """As for the cache itself."""
    s = _state([1, page - 1, page, page + 1, 2 * page + 3], page=page, d=64,
               spare=1, device=device)
    want = oracle(*s)
    _near(paged_attention(*s), want)
    if device == "cuda":
        s2 = _grouped_state([9], [2 * page], [5 * i for i in range(9)],
                            page=page, d=64, nh=8)
        _near(paged_attention(*s2, shared_prefix=_groups([0, 9], [2 * page])),
              oracle(*s2))


def test_pages_are_found_by_a_product():
    """The kernel's division of tokens / 16 below 2^27 by p sixteenths, at
    both sides of every kind of border."""
    for p in list(range(1, 600)) + [1000, 1023, 1025, 65535, 99991,
                                    (1 << 27) // 16 - 1, (1 << 27) - 1]:
        shift = 36 + p.bit_length()
        magic = ((1 << shift) + p - 1) // p
        top = (1 << 27) - 1
        assert top * magic < 1 << 64
        for k in {1, 2, 3, 1000, top // p - 1, top // p}:
            for x in (k * p - 1, k * p, k * p + 1, top):
                if 0 <= x <= top:
                    assert x * magic >> shift == x // p, (x, p)


# ------------------------------------------------- groups and who leads them
@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hold", [
    {0: 0}, {0: 40, 1: 0}, {i: 7 * i % 90 for i in range(69)},
    {i: 320 - 16 * (1 + i % 5) - i % 3 for i in range(70)}])
def test_groups_whose_first_rows_hold_less(hold, d):
    """Empty and short rows in front, whose tables end with them: the others
    see all of their prefix.  In the last case no row holds all of it."""
    q, k, v, tables, lengths = _grouped_state([70], [320], [5] * 70, d=d,
                                              nh=8)
    for i, n in hold.items():
        lengths[i] = n
        tables[i, -(-n // 16):] = -1
    g = _groups([0, 70], [320])
    _near(paged_attention(q, k, v, tables, lengths, shared_prefix=g),
          oracle(q, k, v, tables, lengths))


@gpu
def test_a_group_that_begins_with_padding():
    """Rows without a slot in front of those that have one."""
    q, k, v, tables, lengths = _grouped_state([20], [320], [5] * 20, d=64,
                                              nh=8)
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    slots[:3] = torch.tensor([-1, 99, -1])
    tables[0] = tables[0].flip(0)       # what a clamped number would read
    got = paged_attention(q, k, v, tables, lengths, slots=slots,
                          shared_prefix=_groups([0, 20], [320]))
    want, room = oracle(q[3:], k, v, tables, lengths, slots=slots[3:])
    _near(got[3:], (want, room))
    assert (got[:3] == 0).all()


# --------------------------------------------------------- how work is cut
def _pieces(*args):
    from megatronapp_amd import ops
    if not ops.have_ops():
        pytest.skip("the extension is not built")
    return ops.get_ops().paged_attn_pieces(*args)


@pytest.mark.parametrize("b,groups,max_rows,most,prefix", [
    (3, 2, 2, 20050, 20000), (40, 5, 30, 17000, 16384), (9, 1, 8, 9000, 8192)])
def test_a_long_row_outside_the_group_is_cut(b, groups, max_rows, most,
                                             prefix):
    """A row that shares nothing may be as long as the longest of a group:
    none of its pieces has more than 1024 keys."""
    own, shared, evenly, extra = _pieces(b, 32, 8, 128, most, groups,
                                         max_rows, prefix)
    assert shared > 0 and own * 1024 >= most and evenly <= own
    assert extra >= min(256, own - evenly)
    # rows in general go by what they have of their own
    assert evenly <= max(1, (most - prefix + 255) // 256)


def test_rows_of_one_group_are_cut_by_what_is_their_own():
    for b, own, prefix in ((64, 700, 4096), (256, 1024, 16384)):
        cut = _pieces(b, 32, 8, 128, prefix + own, 1, b, prefix)
        assert cut[0] == cut[2] == 1 < cut[1] and cut[3] == 0


@gpu
def test_a_long_row_beside_a_group():
    own = [3, 70, 20000]
    s = _grouped_state([2, 1], [20000, 0], own, d=128, nh=32, ng=8, page=32)
    _near(paged_attention(*s, shared_prefix=_groups(
        [0, 2, 3], [20000, 0], 2, 20000), max_length=20070), oracle(*s))


def test_pieces_take_a_bounded_room():
    """64 MB for rows' own ones, four times that for all, beyond one of each
    kind; small groups in large batches above all."""
    for b in (3, 200, 512, 2048):
        for nh, ng in ((64, 8), (32, 32), (16, 1)):
            for d in (64, 128):
                row = b * nh * (d + 1) * 4      # of one piece, in bytes
                for groups, rows, prefix in ((0, 1, 0), (1, 4, 32768),
                                             (b, 1, 16384), (1, b, 100000)):
                    own, shared, *_ = _pieces(b, nh, ng, d, prefix + 64,
                                              groups, rows, prefix)
                    assert own == 1 or own * row <= 64 << 20
                    assert (own + shared) * row <= max(256 << 20, 2 * row)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_tables_that_pass_32_bits_are_refused(device):
    for width in (1 << 22, (1 << 22) - 15):
        wide = torch.zeros(2, width, dtype=torch.int32, device=device)
        q, k, v, _, lengths = _state([20, 20], page=512, device=device)
        with pytest.raises(ValueError, match="too long"):
            paged_attention(q, k, v, wide, lengths)
