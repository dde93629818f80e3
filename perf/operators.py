"""Measured cases of the packed attention, the paged attention of single
tokens and the page operators of the cache.

``own`` chooses what ``run`` computes with: the plain forms below (elementary
torch operations in 32 bits, rounded once at the end) or the framework's
operators.  Sequences and rows are given as texts of comma-separated lengths.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# --------------------------------------------------------------------- cases
def listed():
    return [
        # three short prompts admitted in one engine step: latency
        {"name": "prompt, few tokens", "op": "prompt", "type": "bf16",
         "lens": "17,64,9", "tail": 0, "heads": 16, "groups": 16, "dim": 64},
        # a step's waiting prompts packed into one stream, grouped heads;
        # an empty one, a single token, padding behind the last
        {"name": "prompt, ragged", "op": "prompt", "type": "bf16",
         "lens": "801,1,1290,0,333,64,2048,517,129,700", "tail": 37,
         "heads": 32, "groups": 8, "dim": 128},
        # long documents
        {"name": "prompt, long", "op": "prompt", "type": "fp16",
         "lens": "8192,5003,3001,188", "tail": 0, "heads": 32, "groups": 8,
         "dim": 128},
        # a packed training micro-batch, one head for each key head
        {"name": "train, packed", "op": "train", "type": "bf16",
         "lens": "2048,1025,511,1536,77,951,1999,45", "tail": 0,
         "heads": 16, "groups": 16, "dim": 128},
        # many documents of unlike length, grouped heads
        {"name": "train, grouped", "op": "train", "type": "bf16",
         "lens": "2048,1300,257,2047,640,1,1777,900,128,1500,2048,333,1055,"
                 "1280,1006", "tail": 64, "heads": 32, "groups": 8,
         "dim": 64},
        # a few short conversations, nothing shared: latency
        {"name": "decode, few rows", "op": "decode", "type": "bf16",
         "rows": "1,1,1", "prefix": "0,0,0", "own": "41,7,66", "heads": 16,
         "groups": 16, "dim": 64, "page": 16},
        # several system prompts in one batch, one of them unshared
        {"name": "decode, prefix groups", "op": "decode", "type": "fp16",
         "rows": "9,1,6,8", "prefix": "512,0,1040,96",
         "own": "5,190,33,1,250,77,16,140,61,2030,300,12,88,129,1,47,64,201,"
                "9,33,150,74,280,18", "heads": 32, "groups": 8, "dim": 64,
         "page": 16},
        # a batch on one long system prompt
        {"name": "decode, one prefix", "op": "decode", "type": "bf16",
         "rows": "64", "prefix": "4096",
         "own": _text(33 + (i * 211) % 667 for i in range(64)),
         "heads": 32, "groups": 8, "dim": 128, "page": 32},
        # the largest batch on a document that all rows ask about
        {"name": "decode, long prefix", "op": "decode", "type": "bf16",
         "rows": "256", "prefix": "16384",
         "own": _text(1 + (i * 389) % 1024 for i in range(256)),
         "heads": 32, "groups": 8, "dim": 128, "page": 64},
        # one beam search step: every beam continues one of the beams
        {"name": "fork, beams", "op": "fork", "layers": 24, "groups": 16,
         "dim": 64, "page": 16, "pages": 96, "lens": "201,201,201,201",
         "src": "1,1,0,1", "dst": "0,1,2,3"},
        # many samples of one prompt
        {"name": "fork, samples", "op": "fork", "layers": 32, "groups": 8,
         "dim": 128, "page": 64, "pages": 512,
         "lens": _text([8237] + [0] * 63), "src": _text([0] * 63),
         "dst": _text(range(1, 64))},
        # a third of the sequences retire, what is left moves together
        {"name": "retire and compact", "op": "compact", "layers": 16,
         "groups": 8, "dim": 64, "page": 64, "pages": 1500,
         "lens": _text(1 + (i * 977) % 2500 for i in range(64)),
         "free": _text(range(0, 64, 3))},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(
        rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "decode",
                     "decode", "decode", "fork", "compact"])
    heads, groups, dim = rng.choice([(16, 16, 64), (16, 16, 128), (32, 8, 64),
                                     (32, 8, 128)])
    if op in ("prompt", "train"):
        n = _log(rng, 1, 16)
        lens, most = [], _log(rng, 24, 4096 if op == "prompt" else 2048)
        room = 16000
        for _ in range(n):
            lens.append(min(room, rng.randint(0, most)))
            room -= lens[-1]
        lens[rng.randrange(n)] = max(1, min(most, room))
        return {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]),
                "lens": _text(lens), "tail": rng.choice([0, 0, 5, 130]),
                "heads": heads, "groups": groups, "dim": dim}
    page = rng.choice([16, 32, 64])
    if op == "decode":
        total = _log(rng, 1, 200)
        rows, left = [], total
        while left:
            rows.append(min(left, _log(rng, 1, 200)))
            left -= rows[-1]
        longest = _log(rng, 16, 16000)
        prefix = [rng.choice([0, 1, 1]) * rng.randint(0, longest) // page
                  * page for _ in rows]
        most = _log(rng, 1, 1024)
        return {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]),
                "rows": _text(rows), "prefix": _text(prefix),
                "own": _text(rng.randint(1, most) for _ in range(total)),
                "heads": heads, "groups": groups, "dim": dim, "page": page}
    layers = rng.choice([4, 16, 24])
    slots = _log(rng, 2, 48)
    most = _log(rng, 20, 2000)
    lens = [rng.randint(1, most) for _ in range(slots)]
    need = sum(-(-x // page) for x in lens) + slots
    case = {"op": op, "layers": layers, "groups": groups, "dim": dim,
            "page": page, "pages": need + rng.randint(1, 100),
            "lens": _text(lens)}
    some = rng.sample(range(slots), rng.randint(1, slots))
    if op == "fork":
        case["src"] = _text(rng.randrange(slots) for _ in some)
        case["dst"] = _text(some)
    else:
        case["free"] = _text(some)
    return case


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda",
                            dtype=torch.float32) * by).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    op = case["op"]
    if op in ("prompt", "train"):
        t, lens = _TYPES[case["type"]], _ints(case["lens"])
        nh, ng, d = case["heads"], case["groups"], case["dim"]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        total = cu[-1] + case["tail"]
        # keys' scale gives scores of a deviation of 2
        s = {"op": op, "q": normal(total, nh, d, dtype=t, by=2.0),
             "k": normal(total, ng, d, dtype=t),
             "v": normal(total, ng, d, dtype=t), "cu": ints(cu),
             "most": max(lens)}
        if op == "train":
            s["dout"] = normal(total, nh, d, dtype=t)
            for x in "qkv":
                s[x].requires_grad_(True)
        return s
    if op == "decode":
        t, nh, ng = _TYPES[case["type"]], case["heads"], case["groups"]
        d, page = case["dim"], case["page"]
        rows, prefix = _ints(case["rows"]), _ints(case["prefix"])
        mine = _ints(case["own"])
        pages, tables, lengths, at = 0, [], [], 0
        for r, p in zip(rows, prefix):
            shared = list(range(pages, pages + p // page))
            pages += len(shared)
            for n in mine[at:at + r]:
                more = -(-n // page)
                tables.append(shared + list(range(pages, pages + more)))
                lengths.append(p + n)
                pages += more
            at += r
        width = max(len(x) for x in tables)
        # the pool's pages lie in no order
        place = torch.randperm(pages, generator=g, device="cuda").int()
        table = ints([x + [0] * (width - len(x)) for x in tables])
        ends = [0]
        for r in rows:
            ends.append(ends[-1] + r)
        return {"op": op, "q": normal(len(mine), nh, d, dtype=t, by=2.0),
                "k": normal(pages, ng, page, d, dtype=t),
                "v": normal(pages, ng, page, d, dtype=t),
                "tables": place[table.long()], "lengths": ints(lengths),
                "rows": ints(ends), "prefix": ints(prefix),
                "most_rows": max(rows), "most_prefix": max(prefix),
                "most": max(lengths)}
    # the pages of a cache: [layers, 2, pages, groups, page, dim]
    page, lens, pool = case["page"], _ints(case["lens"]), case["pages"]
    place = torch.randperm(pool, generator=g, device="cuda").tolist()
    used, tables = 0, []
    for n in lens:
        more = -(-n // page)
        tables.append(place[used:used + more])
        used += more
    width = max(max(len(x) for x in tables), 1)
    refs = [0] * pool
    for x in tables:
        for p in x:
            refs[p] += 1
    s = {"op": op, "page": page,
         "pages": normal(case["layers"], 2, pool, case["groups"], page,
                         case["dim"], dtype=torch.bfloat16),
         "refs": ints(refs), "lengths": ints(lens),
         "tables": ints([x + [-1] * (width - len(x)) for x in tables])}
    if op == "fork":
        s["src"], s["dst"] = ints(_ints(case["src"])), ints(_ints(case["dst"]))
    else:
        s["free"] = ints(_ints(case["free"]))
        # the scheduler's tables, handed over at the start of each pass
        s["plan"] = tuple(s[x].clone() for x in ("refs", "tables", "lengths"))
    if own:
        from megatronapp_amd.core.inference.paged_kv_cache import PagedKVCache
        s["cache"] = PagedKVCache.from_state(s["pages"], s["refs"],
                                             s["tables"], s["lengths"])
    return s


# --------------------------------------------------------------- plain forms
def _softmax(scores):
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _padded(cu, most, total):
    """Indexes of [sequences, most] places in the stream, which of them
    are in use, and each token's sequence and place."""
    lens = (cu[1:] - cu[:-1]).long()
    at = torch.arange(most, device=cu.device)
    index = (cu[:-1, None].long() + at).clamp(max=max(total - 1, 0))
    token = torch.arange(total, device=cu.device)
    seq = (token[:, None] >= cu[None, 1:]).sum(-1).clamp(max=len(lens) - 1)
    place = (token - cu[:-1].long()[seq]).clamp(0, most - 1)
    return index, at < lens[:, None], seq, place, token < cu[-1]


def _plain_packed(s, dout=None):
    q, k, v, cu, most = s["q"].detach(), s["k"].detach(), s["v"].detach(), \
        s["cu"], s["most"]
    total, nh, d = q.shape
    ng, scale = k.shape[1], 1.0 / math.sqrt(d)
    rep = nh // ng
    index, used, seq, place, live = _padded(cu, most, total)
    n = index.shape[0]

    def heads(x):      # [total, h, d] -> [n, ng, h / ng * most, d]
        return x[index].float().permute(0, 2, 1, 3).reshape(n, ng, -1, d)

    def stream(x, h):  # and back, in the type of the inputs
        x = x.view(n, h, most, d)[seq, :, place]
        return (x * live[:, None, None]).to(q.dtype)

    qf, kf, vf = heads(q), heads(k), heads(v)
    scores = torch.matmul(qf * scale, kf.transpose(2, 3)).view(
        n, ng, rep, most, most)
    later = torch.ones(most, most, dtype=torch.bool, device=q.device).triu(1)
    hide = later | ~used[:, None, :]
    p = _softmax(scores.masked_fill_(hide[:, None, None], -1e30))
    p = p.view(n, ng, rep * most, most)
    out = stream(torch.matmul(p, vf), nh)
    if dout is None:
        return out
    # places behind a sequence's end give nothing
    do = heads(dout) * used[:, None, None, :, None].expand(
        n, ng, rep, most, 1).reshape(n, ng, rep * most, 1)
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, vf.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(2, 3), qf)
    return {"out": out, "dq": stream(dq, nh), "dk": stream(dk, ng),
            "dv": stream(dv, ng)}


def _plain_decode(s):
    q, tables, lengths = s["q"], s["tables"].long(), s["lengths"]
    b, nh, d = q.shape
    ng = s["k"].shape[1]

    def rows(x):       # [pages, ng, page, d] -> [b, ng, tokens, d]
        return x[tables].permute(0, 2, 1, 3, 4).reshape(b, ng, -1, d).float()

    k = rows(s["k"])
    scores = torch.matmul(q.float().view(b, ng, nh // ng, d) / math.sqrt(d),
                          k.transpose(2, 3))
    behind = torch.arange(k.shape[2], device=q.device) >= lengths[:, None]
    p = _softmax(scores.masked_fill(behind[:, None, None], -1e30))
    del k, scores
    return torch.matmul(p, rows(s["v"])).reshape(b, nh, d).to(q.dtype)


def _plain_free(s, slots):
    slots = slots.long()
    rows = s["tables"][slots]
    held = rows >= 0
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(),
                         -held.flatten().int())
    s["tables"][slots] = -1
    s["lengths"][slots] = 0


def _plain_fork(s):
    page = s["page"]
    src, dst = s["src"].long(), s["dst"].long()
    length = s["lengths"][src].long()
    rows = s["tables"][src]
    part = length % page
    copied = (part > 0) & (src != dst)
    free = torch.nonzero(s["refs"] == 0).flatten()
    new = free[(copied.cumsum(0) - 1).clamp(min=0)].int()
    last = (length // page).clamp(max=rows.shape[1] - 1)
    old = rows.gather(1, last[:, None]).flatten()
    rows = rows.scatter(1, last[:, None],
                        torch.where(copied, new, old)[:, None])
    moved = src != dst
    _plain_free(s, dst[moved])
    rows, to = rows[moved], dst[moved]
    s["tables"][to] = rows
    s["lengths"][to] = length[moved].int()
    held = rows >= 0
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(),
                         held.flatten().int())
    frm, to, n = old[copied].long(), new[copied].long(), part[copied]
    token = torch.arange(page, device=n.device) < n[:, None]
    s["pages"][:, :, to] = torch.where(token[:, None, :, None],
                                       s["pages"][:, :, frm],
                                       s["pages"][:, :, to])


def _plain_compact(s):
    live = s["refs"] > 0
    n = live.sum()
    front = torch.arange(live.numel(), device=live.device) < n
    movers = torch.nonzero(live & ~front).flatten()
    holes = torch.nonzero(~live & front).flatten()
    s["pages"][:, :, holes] = s["pages"][:, :, movers]
    to = torch.arange(live.numel(), device=live.device, dtype=torch.int32)
    to[movers] = holes.int()
    s["tables"].copy_(torch.where(s["tables"] >= 0,
                                  to[s["tables"].clamp(min=0).long()],
                                  s["tables"]))
    s["refs"][holes] = s["refs"][movers]
    s["refs"][movers] = 0


# ---------------------------------------------------------------- the passes
def _pool(s):
    """The cache's state; its pages as whole numbers, which have to agree
    in every bit."""
    return {"pages": s["pages"].view(torch.int16), "tables": s["tables"],
            "lengths": s["lengths"], "refs": s["refs"]}


def run(s):
    op = s["op"]
    if not own:
        if op == "prompt":
            return _plain_packed(s)
        if op == "train":
            return _plain_packed(s, s["dout"])
        if op == "decode":
            return _plain_decode(s)
        if op == "fork":
            _plain_fork(s)
        else:
            for x, y in zip(("refs", "tables", "lengths"), s["plan"]):
                s[x].copy_(y)
            _plain_free(s, s["free"])
            _plain_compact(s)
        return _pool(s)
    if op in ("prompt", "train"):
        from megatronapp_amd.core.packed_seq_params import PackedSeqParams
        from megatronapp_amd.core.transformer.packed_attention import (
            packed_attention)
        packing = PackedSeqParams(cu_seqlens_q=s["cu"], cu_seqlens_kv=s["cu"],
                                  max_seqlen_q=s["most"],
                                  max_seqlen_kv=s["most"])
        out = packed_attention(s["q"], s["k"], s["v"], packing)
        if op == "prompt":
            return out
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]),
                                         s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if op == "decode":
        from megatronapp_amd.core.inference.paged_attention import (
            SharedPrefix, paged_attention)
        prefix = SharedPrefix(rows=s["rows"], lengths=s["prefix"],
                              max_rows=s["most_rows"],
                              max_length=s["most_prefix"])
        return paged_attention(s["q"], s["k"], s["v"], s["tables"],
                               s["lengths"], shared_prefix=prefix,
                               max_length=s["most"])
    cache = s["cache"]
    if op == "fork":
        cache.fork(s["src"], s["dst"])
    else:
        cache.load_tables(*s["plan"])
        cache.free(s["free"])
        cache.compact()
    return _pool(s)


def work(case):
    op = case["op"]
    if op in ("prompt", "train"):
        lens = _ints(case["lens"])
        nh, ng, d = case["heads"], case["groups"], case["dim"]
        total = sum(lens) + case["tail"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        if op == "prompt":       # q, k, v read, the output written
            return {"bytes": 2 * total * d * (2 * nh + 2 * ng),
                    "flops": 4 * nh * d * pairs}
        # and its gradient read, three gradients written; five products more
        return {"bytes": 2 * total * d * (4 * nh + 4 * ng),
                "flops": 14 * nh * d * pairs}
    if op == "decode":
        rows, prefix = _ints(case["rows"]), _ints(case["prefix"])
        mine = _ints(case["own"])
        nh, ng, d = case["heads"], case["groups"], case["dim"]
        tokens = sum(mine) + sum(prefix)
        seen = sum(mine) + sum(r * p for r, p in zip(rows, prefix))
        return {"bytes": 4 * tokens * ng * d + 4 * len(mine) * nh * d,
                "flops": 4 * nh * d * seen}
    page, lens = case["page"], _ints(case["lens"])
    token = case["layers"] * 2 * case["groups"] * case["dim"] * 2
    width = max(max(-(-n // page) for n in lens), 1)
    if op == "fork":
        src, dst = _ints(case["src"]), _ints(case["dst"])
        copied = sum(lens[a] % page for a, b in zip(src, dst) if a != b)
        return {"bytes": 2 * copied * token + 4 * case["pages"]
                + 8 * width * len(src), "flops": 0}
    gone = set(_ints(case["free"]))
    left = sum(-(-n // page) for i, n in enumerate(lens) if i not in gone)
    # pages lie in no order: this share of what is left lies behind its end
    moved = left * (case["pages"] - left) / case["pages"]
    return {"bytes": 2 * moved * page * token + 8 * case["pages"]
            + 8 * width * len(lens), "flops": 0}


# ------------------------------------------------------------ from 64 bits
def exact(case, seed):
    op = case["op"]
    if op not in ("prompt", "train", "decode"):
        return None          # moved, not computed
    s = prepare(case, seed)
    q, k, v = (s[x].detach().double() for x in "qkv")
    nh, ng, d = case["heads"], case["groups"], case["dim"]
    rep = nh // ng
    out = torch.zeros_like(q)
    if op == "decode":
        for i, n in enumerate(s["lengths"].tolist()):
            ids = s["tables"][i, :-(-n // case["page"])].long()
            for h in range(ng):
                kk = k[ids, h].reshape(-1, d)[:n]
                vv = v[ids, h].reshape(-1, d)[:n]
                z = (kk @ q[i, h * rep:(h + 1) * rep].t()) / d ** 0.5
                out[i, h * rep:(h + 1) * rep] = torch.softmax(z, 0).t() @ vv
        return out
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    cu = s["cu"].tolist()
    for a, b in zip(cu[:-1], cu[1:]):
        if a == b:
            continue
        ahead = torch.full((b - a, b - a), -math.inf, dtype=torch.float64,
                           device="cuda").triu(1)
        for h in range(nh):
            qq, kk, vv = q[a:b, h], k[a:b, h // rep], v[a:b, h // rep]
            p = torch.softmax(qq @ kk.t() * d ** -0.5 + ahead, -1)
            out[a:b, h] = p @ vv
            if op == "train":
                go = s["dout"][a:b, h].double()
                back = go @ vv.t()
                # the softmax's gradient; its row sums through the output
                back = p * (back - (go * out[a:b, h]).sum(-1, keepdim=True))
                grads[0][a:b, h] = back @ kk * d ** -0.5
                grads[1][a:b, h // rep] += back.t() @ qq * d ** -0.5
                grads[2][a:b, h // rep] += p.t() @ go
    if op == "prompt":
        return out
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
