"""Packed attention against the formula in 64 bits.

Tolerances.  With h = eps / 2 of the type (the most that one rounding is off,
relative to the value), P rounded before the product with V, and O rounded at
the end, |O - ref| <= h |ref| + h P|V|.  dV the same with P^T|dO|.  dS is off
by h |dS|, and by P times what D = sum dO O is off through the rounded O
(|dO| . err(O)); dQ and dK add that through |K| and |Q|, and their own
rounding.  Sums and exponentials are in 32 bits: their share is below 1e-5 of
the terms, far below h = 2^-11, and 5% on top covers it and the products of
errors.  fp16 values below its normal range are off by up to 2^-25.
"""

import math

import pytest
import torch

from megatronapp_amd.core.packed_seq_params import PackedSeqParams
from megatronapp_amd.core.transformer.packed_attention import packed_attention

gpu = pytest.mark.gpu


def _cu(lens, device="cpu"):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def oracle(q, k, v, lens_q, lens_k, causal, scale=None, dout=None, h=0.0,
           tiny=0.0):
    """[t, b, heads, d] -> values in 64 bits and how far a kernel may be
    off: dict of (value, bound)."""
    q, k, v = (x.detach().double() for x in (q, k, v))
    nh, ng, d = q.shape[2], k.shape[2], q.shape[3]
    rep = nh // ng
    scale = d ** -0.5 if scale is None else scale
    names = {"o": q, "dq": q, "dk": k, "dv": k}
    res = {n: [torch.zeros_like(x), torch.zeros_like(x)]
           for n, x in names.items()}
    qa = ka = 0
    for sq, sk in zip(lens_q, lens_k):
        qs, ks = slice(qa, qa + sq), slice(ka, ka + sk)
        qa, ka = qa + sq, ka + sk
        if sq == 0 or sk == 0:
            continue
        see = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril(sk - sq)
        for b in range(q.shape[1]):
            for head in range(nh):
                g = head // rep
                x, y, z = q[qs, b, head], k[ks, b, g], v[ks, b, g]
                s = (x @ y.t() * scale).masked_fill(~see, -math.inf)
                top = s.amax(-1, keepdim=True).clamp(min=-1e300)
                p = torch.exp(s - top)
                p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
                o = p @ z
                err = h * o.abs() + (h * p + tiny) @ z.abs() + tiny
                res["o"][0][qs, b, head] = o
                res["o"][1][qs, b, head] = err
                if dout is None:
                    continue
                do = dout[qs, b, head].double()
                dp = do @ z.t()
                ds = p * (dp - (do * o).sum(-1, keepdim=True))
                # a weight below 2^-126 is zero, and its product too
                lost = 2.0 ** -126 * (dp - (do * o).sum(-1, keepdim=True))
                eds = h * ds.abs() + tiny * see + see * lost.abs() + \
                    p * (do.abs() * err).sum(-1, keepdim=True)
                for n, at, val, e in (
                        ("dq", (qs, b, head), ds @ y, eds @ y.abs()),
                        ("dk", (ks, b, g), ds.t() @ x, eds.t() @ x.abs()),
                        ("dv", (ks, b, g), p.t() @ do / scale,
                         (h * p + tiny * see).t() @ do.abs() / scale)):
                    res[n][0][at] += val * scale
                    res[n][1][at] += e * scale
    for n in ("dq", "dk", "dv"):
        res[n][1] += h * res[n][0].abs() + tiny
    return {n: (a, 1.05 * e) for n, (a, e) in res.items()}


def _rounding(dtype):
    """Half a step, and what is lost at the small end: fp16 has steps of 2^-24
    there, so up to 2^-25; bf16 has the range of 32 bits, in which the kernel's
    exponentials and products are, and those below the smallest normal number,
    2^-126, come out as zero."""
    return (torch.finfo(dtype).eps / 2,
            2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def _inputs(lens_q, lens_k, tail=0, b=1, nh=4, ng=2, d=64,
            dtype=torch.bfloat16, device="cuda", seed=0):
    g = torch.Generator().manual_seed(seed)

    def make(t, heads, by=1.0):
        return (torch.randn(t, b, heads, d, generator=g) * by).to(dtype).to(
            device)
    tq, tk = sum(lens_q) + tail, sum(lens_k) + tail
    return (make(tq, nh, 2.0), make(tk, ng), make(tk, ng), make(tq, nh))


def _near(name, got, want):
    value, bound = want
    off = (got.double() - value).abs() - bound
    assert torch.isfinite(got).all(), name
    assert off.max() <= 0, (name, off.max().item(), got.shape)


def _check(lens_q, lens_k=None, causal=True, grads=True, scale=None, **kw):
    lens_k = lens_q if lens_k is None else lens_k
    q, k, v, dout = _inputs(lens_q, lens_k, **kw)
    dev = q.device
    params = PackedSeqParams(cu_seqlens_q=_cu(lens_q, dev),
                             cu_seqlens_kv=_cu(lens_k, dev))
    for x in (q, k, v):
        x.requires_grad_(grads)
    o = packed_attention(q, k, v, params, causal=causal, softmax_scale=scale)
    h, tiny = _rounding(q.dtype)
    want = oracle(q, k, v, lens_q, lens_k, causal, scale,
                  dout if grads else None, h, tiny)
    _near("o", o.detach(), want["o"])
    assert o.dtype == q.dtype and o.shape == q.shape
    if grads:
        got = torch.autograd.grad(o, (q, k, v), dout)
        for name, x in zip(("dq", "dk", "dv"), got):
            _near(name, x, want[name])
    return o


# ----------------------------------------------------------------- on the CPU
@pytest.mark.parametrize("causal", [True, False])
def test_plain_matches_oracle(causal):
    # in float32 the plain form is within 1e-5 of the terms
    q, k, v, dout = _inputs([5, 0, 1, 9], [5, 3, 4, 2], tail=3, b=2,
                            dtype=torch.float32, device="cpu")
    for x in (q, k, v):
        x.requires_grad_(True)
    lens_q, lens_k = [5, 0, 1, 9], [5, 3, 4, 2]
    o = packed_attention(q, k, v, PackedSeqParams(
        cu_seqlens_q=_cu(lens_q), cu_seqlens_kv=_cu(lens_k)), causal=causal)
    got = (o,) + torch.autograd.grad(o, (q, k, v), dout)
    want = oracle(q, k, v, lens_q, lens_k, causal, None, dout, 1e-5)
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        _near(name, x.detach(), want[name])


def test_plain_gradient_matches_differences():
    q, k, v, _ = _inputs([3, 0, 4], [3, 2, 6], tail=1, nh=2, ng=1, d=4,
                         dtype=torch.float64, device="cpu")
    params = PackedSeqParams(cu_seqlens_q=_cu([3, 0, 4]),
                             cu_seqlens_kv=_cu([3, 2, 6]))
    for x in (q, k, v):
        x.requires_grad_(True)
    assert torch.autograd.gradcheck(
        lambda a, b, c: packed_attention(a, b, c, params), (q, k, v))


def test_plain_three_dims_and_empty_places():
    q, k, v, _ = _inputs([2, 3], [2, 3], tail=4, dtype=torch.float32,
                         device="cpu")
    params = PackedSeqParams(cu_seqlens_q=_cu([2, 3]).long())
    o = packed_attention(q[:, 0], k[:, 0], v[:, 0], params)
    assert o.shape == q[:, 0].shape and (o[5:] == 0).all()
    # ends that run out of the stream are cut off at it
    over = torch.tensor([0, 2, 500], dtype=torch.int32)
    o2 = packed_attention(q[:5, 0], k[:5, 0], v[:5, 0],
                          PackedSeqParams(cu_seqlens_q=over))
    assert torch.equal(o2, o[:5])


@pytest.mark.parametrize("change,message", [
    (dict(q=(4, 4)), "must be"), (dict(k=(4, 3, 8)), "fit"),
    (dict(k=(4, 2, 4), v=(4, 2, 4)), "fit"), (dict(v=(5, 2, 8)), "must be"),
    (dict(kt=torch.float64), "type"), (dict(cu=None), "missing"),
    (dict(cu=torch.zeros(2, 2, dtype=torch.int32)), "cu_seqlens"),
    (dict(cu=torch.zeros(2)), "cu_seqlens"), (dict(scale=0.0), "positive"),
    (dict(scale=-1.0), "positive"), (dict(scale=math.inf), "finite"),
    (dict(cuk=torch.zeros(3, dtype=torch.int32)), "the same"),
])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(change, message, device):
    q = torch.zeros(change.get("q", (4, 4, 8)))
    k = torch.zeros(change.get("k", (4, 2, 8)),
                    dtype=change.get("kt", torch.float32))
    v = torch.zeros(change.get("v", k.shape))
    if k.shape[1] == 3 and "v" not in change:
        v = torch.zeros(k.shape)
    cu = change["cu"] if "cu" in change else _cu([4])
    cuk = change.get("cuk", cu)
    if device == "cuda":
        q, k, v = (x.cuda() for x in (q, k, v))
        cu, cuk = (x if x is None else x.cuda() for x in (cu, cuk))
    params = PackedSeqParams(cu_seqlens_q=cu, cu_seqlens_kv=cuk)
    with pytest.raises(ValueError, match=message):
        packed_attention(q, k, v, params, softmax_scale=change.get("scale"))


# ----------------------------------------------------------------- on the GPU
@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [
    [1], [2, 1, 3], [31, 32, 33], [64, 65, 63], [127, 128, 129], [257, 511],
    [0, 5, 0, 300, 1, 0]])
def test_lengths(lens, dtype, d):
    _check(lens, dtype=dtype, d=d, tail=len(lens) % 3)


@gpu
@pytest.mark.parametrize("nh,ng", [(1, 1), (6, 6), (8, 1), (6, 2), (32, 8)])
def test_head_layouts(nh, ng):
    _check([70, 3, 190], nh=nh, ng=ng, d=128, tail=130)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q,lens_k", [
    ([5, 64, 1], [200, 64, 77]), ([130, 9], [129, 300]),
    ([90, 200, 7], [10, 0, 3]), ([0, 4], [50, 4])])
def test_queries_and_keys_of_other_lengths(lens_q, lens_k, causal):
    _check(lens_q, lens_k, causal=causal, d=64)
    _check(lens_q, lens_k, causal=causal, d=128, tail=9)


@gpu
def test_batch_and_scale():
    _check([40, 0, 100], b=3, d=64, scale=0.31)
    _check([40, 0, 100], b=2, d=128, causal=False, scale=0.05)


@gpu
@pytest.mark.parametrize("lens,nh,ng,d,b", [
    ([300], 8, 1, 64, 1),               # four shares of a tile's work
    ([700, 20, 100], 16, 1, 128, 1),    # eight, some without any
    ([600], 3, 1, 128, 2),
    ([40] * 20, 32, 1, 128, 1),         # more tiles than the host expects
    ([2100], 2, 2, 128, 1),             # of one head
])
def test_shares_of_the_keys_gradients(lens, nh, ng, d, b):
    """Few tiles: several blocks share the queries of one."""
    _check(lens, nh=nh, ng=ng, d=d, b=b, tail=5)
    _check(lens, nh=nh, ng=ng, d=d, b=b, causal=False,
           dtype=torch.float16)


@gpu
def test_shares_without_queries():
    _check([0, 300], [50, 300], nh=8, ng=1, d=64)
    _check([300, 7], [40, 0], nh=16, ng=1, d=128)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens_q,lens_k,causal", [
    ([513], None, True),
    ([1100], None, False),
    ([700, 0, 900], None, True),
    ([5], [1500], True),                # of two halves the queries see both
    ([40, 3], [63, 1200], True),        # and here the first one alone
    ([1300], [600], True),              # rows without keys
])
def test_two_halves_of_the_keys(lens_q, lens_k, causal, d):
    """Few tiles of long sequences: eight waves a tile."""
    _check(lens_q, lens_k, causal=causal, d=d, nh=2, ng=1, tail=3,
           dtype=torch.float16)
    _check(lens_q, lens_k, causal=causal, d=d, nh=3, ng=3, grads=False)
    # scores of some 20: all weight on few keys, in one half or the other
    _check(lens_q, lens_k, causal=causal, d=d, nh=1, ng=1, scale=1.0)


@gpu
@pytest.mark.parametrize("lens,heads", [
    ([7 * i % 23 for i in range(60)], 32),
    ([300, 513, 1, 129] + [40] * 50, 16),
])
def test_many_tiles(lens, heads):
    """Blocks of four waves for the gradients of the keys."""
    _check(lens, nh=heads, ng=heads, d=64, tail=9)
    _check(lens, nh=heads, ng=heads, d=64, causal=False)


@gpu
def test_many_sequences():
    _check([(i * 7) % 13 for i in range(300)], nh=2, ng=1, d=64, tail=2)


@gpu
def test_long_sequence():
    _check([2100, 700], nh=2, ng=1, d=128)


@gpu
def test_large_scores_and_infinite_keys():
    q, k, v, _ = _inputs([100], [100], d=64)
    k = k * 60.0        # scores of some hundreds: one key takes all
    cu = PackedSeqParams(cu_seqlens_q=_cu([100], "cuda"))
    o = packed_attention(q, k, v, cu)
    h, tiny = _rounding(q.dtype)
    _near("o", o, oracle(q, k, v, [100], [100], True, h=h)["o"])


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_sequences_do_not_meet(d):
    """NaN and infinities of other sequences and behind the last one change
    nothing, forward and backward."""
    lens = [40, 100, 33]
    q, k, v, dout = _inputs(lens, lens, tail=50, d=d)
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))

    def run(q, k, v, dout):
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = packed_attention(*x, params)
        return (o.detach(),) + torch.autograd.grad(o, x, dout)

    want = run(q, k, v, dout)
    for t in (q, k, v, dout):
        t[40:140] = math.nan
        t[173:] = math.inf
        t[180:] = math.nan
    for name, a, b in zip(("o", "dq", "dk", "dv"), run(q, k, v, dout), want):
        assert torch.equal(a[:40], b[:40]) and \
            torch.equal(a[140:173], b[140:173]), name
        assert (a[173:] == 0).all(), name


@gpu
def test_views_broadcast_and_strided_gradient():
    """Parts of one fused projection, a key head expanded over heads, and an
    output gradient that is no plain tensor."""
    lens = [50, 77]
    t, nh, d = sum(lens), 4, 64
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(t, 2, nh, 3 * d, generator=g).bfloat16().cuda()
    q, k, v = fused[..., :d], fused[..., d:2 * d], fused[..., 2 * d:]
    one = torch.randn(t, 2, 1, d, generator=g).bfloat16().cuda()
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))
    h, tiny = _rounding(torch.bfloat16)
    wide = torch.randn(2, nh, t, d, generator=g).bfloat16().cuda()
    dout = wide.permute(2, 0, 1, 3)
    for kk in (k, one.expand(t, 2, nh, d)):
        x = [u.detach().requires_grad_(True) for u in (q, kk, v)]
        o = packed_attention(*x, params)
        want = oracle(*x, lens, lens, True, None, dout, h)
        _near("o", o.detach(), want["o"])
        for name, u in zip(("dq", "dk", "dv"),
                           torch.autograd.grad(o, x, dout)):
            _near(name, u, want[name])
    # rows that start off 16 bytes are laid out first
    odd = torch.empty(t * 2 * nh * d + 1, dtype=torch.bfloat16,
                      device="cuda")[1:].view(t, 2, nh, d)
    odd.copy_(q)
    assert torch.equal(packed_attention(odd, k, v, params),
                       packed_attention(q, k, v, params))
    # the gradient of a sum is an expanded scalar
    x = [u.detach().clone().requires_grad_(True) for u in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*x, params).sum(), x)
    want = oracle(*x, lens, lens, True, None,
                  torch.ones_like(dout), h)
    for name, u in zip(("dq", "dk", "dv"), got):
        _near(name, u, want[name])


@gpu
def test_rows_far_apart():
    """Offsets past 2^31 elements."""
    lens, step = [40, 30], 1 << 25
    store = torch.zeros(70 * step + 256, dtype=torch.bfloat16, device="cuda")
    q, k, v, _ = _inputs(lens, lens, nh=2, ng=1, d=64)
    far = torch.as_strided(store, (70, 1, 2, 64), (step, 128, 64, 1))
    far.copy_(q)
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))
    assert torch.equal(packed_attention(far, k, v, params),
                       packed_attention(q, k, v, params))


@gpu
def test_same_bits_twice_and_on_another_stream():
    lens = [300, 41, 200]
    q, k, v, dout = _inputs(lens, lens, d=128)
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))

    def run():
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = packed_attention(*x, params)
        return (o.detach(),) + torch.autograd.grad(o, x, dout)

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@gpu
def test_captured_and_replayed():
    """Forward and backward in a graph; new lengths and values in the same
    tensors take effect on replay."""
    lens = [100, 28, 64]
    q, k, v, dout = _inputs(lens, lens, d=64)
    cu = _cu(lens, "cuda")
    params = PackedSeqParams(cu_seqlens_q=cu)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def run():
        o = packed_attention(*x, params)
        return (o.detach(),) + torch.autograd.grad(o, x, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for new in ([100, 28, 64], [1, 190, 1], [64, 64, 60], [0, 0, 192]):
        cu.copy_(_cu(new))
        with torch.no_grad():
            x[0].mul_(0.9)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, run()):
            assert torch.equal(a, b), new


@gpu
def test_shares_captured_and_replayed():
    """The shares are chosen when the graph is made; later lengths are cut as
    these were, and two graphs keep their sums apart."""
    lens = [700, 20, 100]
    q, k, v, dout = _inputs(lens, lens, nh=16, ng=1, d=128)
    cu = _cu(lens, "cuda")
    params = PackedSeqParams(cu_seqlens_q=cu)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def run():
        o = packed_attention(*x, params)
        return (o.detach(),) + torch.autograd.grad(o, x, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(run())
    for new in (lens, [1, 818, 1], [0, 0, 820], [300, 300, 220]):
        cu.copy_(_cu(new))
        graphs[0].replay()
        graphs[1].replay()
        want = run()
        graphs[0].replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), new


@gpu
def test_gradient_matches_differences():
    """The kernel's gradient against central differences of the formula in
    64 bits, along one direction for each input.  The differences' own error
    (step^2 times a third derivative of order one) is below 1e-5 of them."""
    lens = [33, 70]
    q, k, v, dout = _inputs(lens, lens, d=64)
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*x, params), x, dout)
    h, _ = _rounding(q.dtype)
    want = oracle(q, k, v, lens, lens, True, None, dout, h)
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(x[i].shape, generator=g).double().cuda()
        loss = []
        for step in (1e-4, -1e-4):
            y = [t.double() for t in (q, k, v)]
            y[i] = y[i] + step * way
            o = oracle(*y, lens, lens, True)["o"][0]
            loss.append((o * dout.double()).sum())
        slope = (loss[0] - loss[1]) / 2e-4
        along = (got[i].double() * way).sum()
        room = (want[name][1] * way.abs()).sum() + 1e-5 * slope.abs()
        assert (along - slope).abs() <= room, (name, along, slope)


@gpu
def test_refusals_on_the_gpu():
    params = PackedSeqParams(cu_seqlens_q=_cu([4], "cuda"))
    for shape, dtype in (((4, 2, 32), torch.bfloat16),
                         ((4, 2, 64), torch.float32)):
        x = torch.zeros(shape, dtype=dtype, device="cuda")
        with pytest.raises(ValueError, match="head size"):
            packed_attention(x, x, x, params)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="device"):
        packed_attention(x, x.cpu(), x, params)
    with pytest.raises(ValueError, match="device"):
        packed_attention(x, x, x, PackedSeqParams(cu_seqlens_q=_cu([4])))
    empty = x[:0]
    assert packed_attention(empty, empty, empty, params).shape == (0, 2, 64)
    with pytest.raises(ValueError, match="must be"):
        packed_attention(x[0, 0, 0], x, x, params)
    # no queries, or no heads of them: nothing for the keys, and no keys:
    # nothing for the queries
    for q, k in ((empty, x), (x[:, :0], x), (x, empty)):
        q, k, v = (t.clone().requires_grad_(True) for t in (q, k, k))
        o = packed_attention(q, k, v, params)
        assert o.shape == q.shape and (o == 0).all()
        for t, g in zip((q, k, v), torch.autograd.grad(o.sum(), (q, k, v))):
            assert g.shape == t.shape and (g == 0).all()


@gpu
def test_no_second_gradient():
    q, k, v, dout = _inputs([5], [5])
    params = PackedSeqParams(cu_seqlens_q=_cu([5], q.device))
    q.requires_grad_()
    o = packed_attention(q, k, v, params)
    with pytest.raises(RuntimeError, match="gradient"):
        torch.autograd.grad(o, q, dout, create_graph=True)
    o = packed_attention(q, k, v, params)
    with torch.no_grad():
        q.add_(1)                       # the backward needs it as it was
    with pytest.raises(RuntimeError, match="modified"):
        o.backward(dout)


@gpu
def test_flash_attention_keeps_sequences_apart():
    """The layers' attention hands a packed stream to the kernel, and gives
    what the eager path gives."""
    from tests.utils import destroy, initialize_model_parallel
    from megatronapp_amd.core.enums import AttnMaskType
    from megatronapp_amd.core.transformer.dot_product_attention import (
        DotProductAttention, FlashAttention)
    from megatronapp_amd.core.transformer_config import TransformerConfig
    initialize_model_parallel()
    cfg = TransformerConfig(num_layers=1, hidden_size=256,
                            num_attention_heads=4, num_query_groups=2,
                            bf16=True, hidden_dropout=0.0,
                            attention_dropout=0.0)
    lens = [100, 28, 128]
    q, k, v, _ = _inputs(lens, lens, d=64)
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"),
                             cu_seqlens_kv=_cu(lens, "cuda"))
    h, _ = _rounding(q.dtype)
    want = oracle(q, k, v, lens, lens, True, h=h)["o"]
    got = FlashAttention(cfg, 1, AttnMaskType.causal)(
        q, k, v, packed_seq_params=params)
    assert got.shape == (256, 1, 256)
    _near("flash", got.view(q.shape), want)
    # the eager path rounds the scores too (relative to the largest, here
    # below 16: off by 16 h in the exponent)
    eager = DotProductAttention(cfg, 1, AttnMaskType.causal)(
        q.float(), k.float(), v.float(), packed_seq_params=params)
    _near("eager", eager.view(q.shape), want)
    destroy()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_padding_causal_is_causal_in_a_packed_stream(device):
    from tests.utils import destroy, initialize_model_parallel
    from megatronapp_amd.core.enums import AttnMaskType
    from megatronapp_amd.core.transformer.dot_product_attention import (
        FlashAttention)
    from megatronapp_amd.core.transformer_config import TransformerConfig
    initialize_model_parallel()
    cfg = TransformerConfig(num_layers=1, hidden_size=256,
                            num_attention_heads=4, num_query_groups=2,
                            bf16=device == "cuda", hidden_dropout=0.0,
                            attention_dropout=0.0)
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    q, k, v, _ = _inputs([10, 6], [10, 6], dtype=dtype, device=device)
    params = PackedSeqParams(cu_seqlens_q=_cu([10, 6], device),
                             cu_seqlens_kv=_cu([10, 6], device))
    got = [FlashAttention(cfg, 1, t)(q, k, v, packed_seq_params=params)
           for t in (AttnMaskType.causal, AttnMaskType.padding_causal,
                     AttnMaskType.padding)]
    assert torch.equal(got[0], got[1])
    assert not torch.equal(got[0], got[2])
    destroy()


def _off_16_bytes(x):
    """The same values, contiguous, from two bytes behind a border on."""
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(
        x.shape)
    assert y.is_contiguous() and y.data_ptr() % 16 == 2
    return y.copy_(x.detach())


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_contiguous_tensors_off_16_bytes(d):
    """All four inputs, which the kernels load 16 bytes at a time."""
    lens = [50, 0, 177]
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))

    def run(x):
        x = [t.detach().requires_grad_(i < 3) for i, t in enumerate(x)]
        o = packed_attention(*x[:3], params)
        return (o.detach(),) + torch.autograd.grad(o, x[:3], x[3])

    inputs = _inputs(lens, lens, tail=3, d=d)
    for a, b in zip(run(inputs), run([_off_16_bytes(t) for t in inputs])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("mask", ["causal", "padding"])
@pytest.mark.parametrize("cu_q,cu_k,tq,tk", [
    ([3, 10, 20], None, 20, 20),            # places in front
    ([0, 10, 16], None, 20, 20),            # and behind
    ([0, 10, 20, 20], None, 20, 20),        # an empty last one
    ([2, 2, 9, 9, 15], None, 18, 18),       # all of these
    ([0, 4, 4, 9], [0, 7, 10, 12], 9, 12),  # continued prompts, one empty
    ([1, 6, 8], [3, 5, 5], 10, 7),          # rows and sequences without keys
    ([0, 5, 500], None, 12, 12),            # an end out of the stream
    ([4], None, 6, 6),                      # no sequence at all
])
def test_fallback_gives_what_the_kernel_gives(cu_q, cu_k, tq, tk, mask,
                                              device):
    """32 bits are not the kernel's, so the layers' attention takes the eager
    path; both are off by some 1e-6 of terms of order one."""
    from tests.utils import destroy, initialize_model_parallel
    from megatronapp_amd.core.enums import AttnMaskType
    from megatronapp_amd.core.transformer.dot_product_attention import (
        FlashAttention)
    from megatronapp_amd.core.transformer_config import TransformerConfig
    initialize_model_parallel()
    cfg = TransformerConfig(num_layers=1, hidden_size=32,
                            num_attention_heads=4, num_query_groups=2,
                            hidden_dropout=0.0, attention_dropout=0.0)
    g = torch.Generator().manual_seed(8)
    q, dout = (torch.randn(tq, 2, 4, 8, generator=g).to(device)
               for _ in range(2))
    k, v = (torch.randn(tk, 2, 2, 8, generator=g).to(device)
            for _ in range(2))
    x = [t.requires_grad_(True) for t in (q, k, v)]
    params = PackedSeqParams(*(
        ["thd"] + [c if c is None else
                   torch.tensor(c, dtype=torch.int32, device=device)
                   for c in (cu_q, cu_k)]))
    got = FlashAttention(cfg, 1, AttnMaskType[mask])(
        *x, packed_seq_params=params).view(tq, 2, 4, 8)
    on_host = PackedSeqParams(*(
        ["thd"] + [c if c is None else torch.tensor(c) for c in (cu_q, cu_k)]))
    y = [t.detach().cpu().requires_grad_(True) for t in x]
    want = packed_attention(*y, on_host, causal=mask == "causal")
    pairs = [(got, want)] + list(zip(
        torch.autograd.grad(got, x, dout),
        torch.autograd.grad(want, y, dout.cpu(), materialize_grads=True,
                            allow_unused=True)
        if want.requires_grad else [torch.zeros_like(t) for t in y]))
    for a, b in pairs:
        assert (a.detach().cpu() - b.detach()).abs().max() < 1e-5
    destroy()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_has_its_derivative_or_is_refused(which, device):
    """On the CPU the tangent is that of differences; the kernel has none, and
    says so rather than give a constant."""
    from torch.autograd import forward_ad
    dtype = torch.bfloat16 if device == "cuda" else torch.float64
    q, k, v, dout = _inputs([5, 3], [5, 3], device=device, dtype=dtype)
    x, way = [q, k, v], [dout, k.flip(0), v.flip(0)][which]
    params = PackedSeqParams(cu_seqlens_q=_cu([5, 3], device))
    for wants in (False, True):     # a reverse gradient beside it
        y = [t.clone().requires_grad_(wants) for t in x]
        with forward_ad.dual_level():
            y[which] = forward_ad.make_dual(y[which], way)
            if device == "cuda":
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    packed_attention(*y, params)
                continue
            got = forward_ad.unpack_dual(packed_attention(*y, params)).tangent
        ends = []
        for step in (1e-5, -1e-5):
            z = list(x)
            z[which] = z[which] + step * way
            ends.append(packed_attention(*z, params))
        # the third derivative, of some hundreds at most, times the step's
        # square, and 64 bits' 1e-16 of values of order one over the step
        assert (got - (ends[0] - ends[1]) / 2e-5).abs().max() < 1e-7
    if device == "cuda":            # without a wish for it, a value
        with forward_ad.dual_level(), forward_ad._set_fwd_grad_enabled(False):
            y[which] = forward_ad.make_dual(x[which], way)
            packed_attention(*y, params)


@gpu
@pytest.mark.parametrize("lens", [[300, 41, 200], [2100], [64, 1000, 3]])
@pytest.mark.parametrize("d", [64, 128])
def test_the_same_bits_with_and_without_gradients(lens, d):
    """Recomputation runs the first forward without them and the second one
    with them.  Large scores: the running maximum moves often."""
    q, k, v, _ = _inputs(lens, lens, d=d)
    q = q * 6.0
    params = PackedSeqParams(cu_seqlens_q=_cu(lens, "cuda"))
    with torch.no_grad():
        first = packed_attention(q, k, v, params)
    again = packed_attention(q.requires_grad_(True), k, v, params)
    assert torch.equal(first, again.detach())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_scores_of_a_packed_stream_are_reported(device):
    """A tracer that asks for them gets them: the kernel has none."""
    from tests.utils import destroy, initialize_model_parallel
    from megatronapp_amd.core.enums import AttnMaskType
    from megatronapp_amd.core.tensor_tracer import (FlagType,
                                                    enable_tensor_tracers)
    from megatronapp_amd.core.transformer.dot_product_attention import (
        FlashAttention)
    from megatronapp_amd.core.transformer_config import TransformerConfig
    initialize_model_parallel()
    dtype = torch.float16 if device == "cuda" else torch.float32
    cfg = TransformerConfig(num_layers=1, hidden_size=256,
                            num_attention_heads=4, num_query_groups=2,
                            fp16=device == "cuda", hidden_dropout=0.0,
                            attention_dropout=0.0)
    q, k, v, _ = _inputs([10, 6], [10, 6], dtype=dtype, device=device)
    cu = _cu([10, 6], device)
    attend = FlashAttention(cfg, 1, AttnMaskType.causal)
    tt, seen = enable_tensor_tracers(), []
    tt.set_num_layers(1)
    tt.set_report(seen.append)
    for asked in ("False", "True"):
        tt.tt_flags.set_by_configs({"Raw_attention_score": asked})
        o = attend(q, k, v, packed_seq_params=PackedSeqParams(
            cu_seqlens_q=cu, cu_seqlens_kv=cu))
        assert o.shape == (16, 1, 256)
        assert len(seen) == (asked == "True")
    tt.set_report(None)
    assert seen[0]["update_type"] == FlagType.RawAttentionScore.value
    assert seen[0]["args"] == [1, 4, 16, 16]
    p = torch.tensor(seen[0]["result"]).view(4, 16, 16)
    assert (p[:, 10:, :10] == 0).all() and (p.triu(1) == 0).all()
    destroy()


def test_shares_take_a_bounded_room():
    """134 MB at most, also where sequences are short and each has a tile."""
    from megatronapp_amd import ops
    if not ops.have_ops():
        pytest.skip("the extension is not built")
    shares_of = ops.get_ops().packed_attn_shares
    assert shares_of(1, 4096, 4096, 1, 32, 8, 128)[0] == 2
    most = 0
    for n in (1, 2, 8, 40):
        for t in (1, 256, 1024, 8192):
            for rep in (1, 4, 16, 64):
                for heads in (1, 8, 32, 64, 96, 200):
                    for d in (64, 128):
                        shares, floats = shares_of(n, t, t, 1, heads * rep,
                                                   heads, d)
                        assert (floats == 0) == (shares == 1)
                        most = max(most, 4 * floats)
    assert 100e6 < most < 135e6


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_ends_behind_32_bits(device):
    """They run out of the stream like any other that does."""
    q, k, v, _ = _inputs([40], [40], device=device)

    def run(*cu):
        return packed_attention(q, k, v, PackedSeqParams(
            cu_seqlens_q=torch.tensor(cu, device=device)))

    assert torch.equal(run(0, 5, (1 << 32) + 7), run(0, 5, 40))
    assert torch.equal(run(-(1 << 32) + 3, 5, 9), run(0, 5, 9))
