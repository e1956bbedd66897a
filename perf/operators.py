"""The operators of beam search over a shared prompt, in their plain form (torch)
and as the framework's calls: what is measured, on which inputs.

attention   attention_decode_shared: one new token per row, rows in groups
            whose sequences hold the same leading cache pages
append      qk_norm_rope_kv_append_batch: new tokens of several sequences,
            normalised, rotated and stored in the paged cache
select      beam_select: the best continuations over beams x vocabulary
reorder     KVCache.reorder: the beams' caches follow the chosen parents

Shapes are those of the repository's model configurations (16 or 32 query
heads over 8 KV heads, head dims 64 and 128, vocabularies 32000, 128256 and
151936) and generic ones around them.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # four beams of a short prompt, early in the answer: latency
        dict(name="attention-beams4-p512", op="attention", groups=1, rows=4, prefix=512, suffix=20,
             heads=16, kv=8, hd=128, page=16, window=0),
        # eight beams of a long prompt, well into the answer, 64-wide heads
        dict(name="attention-beams8-p2048", op="attention", groups=1, rows=8, prefix=2048,
             suffix=150, heads=32, kv=8, hd=64, page=32, window=0),
        # 32 users behind one system prompt, answers of uneven length
        dict(name="attention-users32-p2048", op="attention", groups=1, rows=32, prefix=2048,
             suffix=600, heads=32, kv=8, hd=128, page=16, window=0),
        # seven prompts with five beams each, uneven prompts, a page size that divides nothing
        dict(name="attention-groups7x5-odd", op="attention", groups=7, rows=5, prefix=1001,
             suffix=77, heads=16, kv=8, hd=128, page=24, window=0),
        # 64 samples of one very long document
        dict(name="attention-samples64-p32768", op="attention", groups=1, rows=64, prefix=32768,
             suffix=64, heads=32, kv=8, hd=128, page=64, window=0),
        # one decode step's append for 32 sequences
        dict(name="append-32x1", op="append", seqs=32, tokens=1, heads=32, kv=8, hd=128, page=16,
             norm=False),
        # prompts of uneven length taken in together, heads with their own norm
        dict(name="append-7-prompts", op="append", seqs=7, tokens=1200, heads=16, kv=8, hd=128,
             page=24, norm=True),
        # one request, four beams, a small vocabulary: latency
        dict(name="select-4x32000", op="select", groups=1, beams=4, vocab=32000, k=4, done=0),
        # eight beams, the largest vocabulary, twice as many candidates as beams
        dict(name="select-8x151936", op="select", groups=1, beams=8, vocab=151936, k=16, done=1),
        # a batch of requests
        dict(name="select-32x5x128256", op="select", groups=32, beams=5, vocab=128256, k=10,
             done=20),
        # one request's beams after a step
        dict(name="reorder-4", op="reorder", groups=1, beams=4, layers=16, kv=8, hd=64, page=16,
             length=525, keep=2),
        # a batch of requests, large pages
        dict(name="reorder-4x8", op="reorder", groups=4, beams=8, layers=28, kv=8, hd=128,
             page=32, length=316, keep=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "select", "reorder"])
    if op == "attention":
        while True:
            c = dict(op=op, groups=rng.choice([1, 1, 1, 2, 3, 6]), rows=_log(rng, 2, 64),
                     prefix=_log(rng, 16, 32768), suffix=_log(rng, 1, 1000),
                     kv=rng.choice([1, 2, 4, 8]), hd=rng.choice([64, 128, 128, 32, 96]),
                     page=rng.choice([16, 32, 64, 5, 24, 128]),
                     window=rng.choice([0, 0, 0, 0, 700]))
            c["heads"] = c["kv"] * rng.choice([1, 2, 4, 8, 3])
            n = c["groups"] * c["rows"]
            if n <= 64 and n * c["heads"] * c["hd"] * (c["prefix"] + c["suffix"]) <= 64 * 32 * 128 * 32832 \
                    and c["kv"] * c["hd"] * (c["groups"] * c["prefix"] + n * c["suffix"]) <= 8 * 128 * 36000:
                return c
    if op == "append":
        kv = rng.choice([1, 2, 4, 8])
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, tokens=_log(rng, 1, max(1, 4000 // seqs)),
                    heads=kv * rng.choice([1, 2, 4, 3]), kv=kv, hd=rng.choice([64, 128, 32, 96]),
                    page=rng.choice([16, 32, 64, 5]), norm=rng.random() < 0.5)
    if op == "select":
        while True:
            g, b, v = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), _log(rng, 500, 160000)
            if g * b * v <= 32 * 5 * 128256:
                return dict(op=op, groups=g, beams=b, vocab=v, k=b * rng.choice([1, 2]),
                            done=rng.randint(0, g * b // 3))
    while True:
        b = rng.choice([2, 3, 4, 5, 8])
        c = dict(op=op, groups=_log(rng, 1, 12), beams=b, layers=_log(rng, 1, 28),
                 kv=rng.choice([1, 2, 4, 8]), hd=rng.choice([64, 128, 32]),
                 page=rng.choice([1, 8, 16, 32, 5]), length=_log(rng, 3, 700),
                 keep=rng.randint(1, b))
        if c["groups"] * b * c["length"] * c["layers"] * c["kv"] * c["hd"] <= 4 * 8 * 316 * 28 * 1024:
            return c


# ---------------------------------------------------------------------------
# layouts that follow from a case alone
# ---------------------------------------------------------------------------
def _lengths(c):
    """attention: ([prefix of each group], [positions behind the prefix of each row]), the
    first of each at the case's largest."""
    r = random.Random(str(sorted((k, v) for k, v in c.items() if k != "name")))
    pre = [c["prefix"] if g == 0 else max(1, int(c["prefix"] * r.uniform(0.3, 1.0)))
           for g in range(c["groups"])]
    suf = [c["suffix"] if i == 0 else r.randint(0, c["suffix"])
           for i in range(c["groups"] * c["rows"])]
    return pre, suf


def _counts(c):
    """append: ([positions held], [new tokens]) of each sequence."""
    r = random.Random(str(sorted((k, v) for k, v in c.items() if k != "name")))
    held = [r.randint(0, 100) for _ in range(c["seqs"])]
    new = [c["tokens"] if i == 0 else max(1, int(c["tokens"] * r.uniform(0.2, 1.0)))
           for i in range(c["seqs"])]
    return held, new


class _Pages:
    """Page tables as the cache hands pages out: in order, the next one each time."""

    def __init__(self, page):
        self.page, self.next, self.rows = page, 0, []

    def grow(self, row, length):
        while len(row) * self.page < length:
            row.append(self.next)
            self.next += 1

    def fork(self, src, length):
        row = list(src[:length // self.page])
        if length % self.page:
            row.append(self.next)
            self.next += 1
        return row

    def table(self, device):
        n = max(len(r) for r in self.rows)
        return torch.tensor([r + [0] * (n - len(r)) for r in self.rows], device=device)


def _rope(max_pos, hd, device):
    """Position tables [max_pos, hd/2], angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
    a = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_attention(c, seed):
    g, dev = _gen(seed), "cuda"
    pre, suf = _lengths(c)
    pt, rows, n = _Pages(c["page"]), c["rows"], c["groups"] * c["rows"]
    tails = []
    for gi, p in enumerate(pre):
        first = []
        pt.grow(first, p)
        pt.rows.append(first)
        for _ in range(rows - 1):
            pt.rows.append(pt.fork(first, p))
            if p % c["page"]:
                tails.append((first[-1], pt.rows[-1][-1]))
    lens = [pre[i // rows] + suf[i] for i in range(n)]
    for i in range(n):
        pt.grow(pt.rows[i], lens[i])
    held = pt.next
    for i in range(n):
        pt.grow(pt.rows[i], lens[i] + 1)
    shape = (pt.next, c["page"], c["kv"], c["hd"])
    kp = torch.randn(shape, generator=g, device=dev)
    vp = torch.randn(shape, generator=g, device=dev)
    for a, b in tails:
        kp[b] = kp[a]
        vp[b] = vp[a]
    qkv = torch.randn(n, (c["heads"] + 2 * c["kv"]) * c["hd"], generator=g, device=dev)
    qkv[:, :c["heads"] * c["hd"]] *= 2.0
    top = max(max(lens) + 1, c["page"])
    cos, sin = _rope(top, c["hd"], dev)
    st = dict(c=c, k=kp, v=vp, qkv=qkv, cos=cos, sin=sin, table=pt.table(dev),
              lens=torch.tensor(lens, device=dev), pre=torch.tensor(pre, device=dev),
              pmax=max(pre), smax=max(suf) + 1)
    if own:
        import synapse_b200 as sb
        ctx = sb.Context(torch.cuda.current_device())
        cache = sb.KVCache(ctx, top, c["kv"], c["hd"], 1, n, c["page"], pt.next)
        for gi, p in enumerate(pre):
            cache.advance(p, gi * rows)
            for j in range(1, rows):
                cache.fork(gi * rows, gi * rows + j, p)
        for i in range(n):
            cache.advance(suf[i], i)
        assert cache.pages_free() == pt.next - held
        pools = cache.pages(0)
        pools[0].copy_(kp)
        pools[1].copy_(vp)
        plan = sb.DecodePlan(cache, c["heads"])
        plan.set([list(range(gi * rows, (gi + 1) * rows)) for gi in range(c["groups"])])
        st.update(ctx=ctx, cache=cache, pools=pools, plan=plan)
    return st


def _prepare_append(c, seed):
    g, dev = _gen(seed), "cuda"
    held, new = _counts(c)
    pt = _Pages(c["page"])
    for i in range(c["seqs"]):
        pt.rows.append([])
        pt.grow(pt.rows[i], held[i])
    for i in range(c["seqs"]):
        pt.grow(pt.rows[i], held[i] + new[i])
    shape = (pt.next, c["page"], c["kv"], c["hd"])
    kp = torch.randn(shape, generator=g, device=dev)
    vp = torch.randn(shape, generator=g, device=dev)
    qkv = torch.randn(sum(new), (c["heads"] + 2 * c["kv"]) * c["hd"], generator=g, device=dev)
    qn = kn = None
    if c["norm"]:
        qn = 1 + 0.1 * torch.randn(c["hd"], generator=g, device=dev)
        kn = 1 + 0.1 * torch.randn(c["hd"], generator=g, device=dev)
    top = max([c["page"]] + [h + t for h, t in zip(held, new)])
    cos, sin = _rope(top, c["hd"], dev)
    seq = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(new)).to(dev)
    pos = torch.cat([torch.arange(h, h + t) for h, t in zip(held, new)]).to(dev)
    st = dict(c=c, k=kp, v=vp, qkv=qkv, qn=qn, kn=kn, cos=cos, sin=sin, table=pt.table(dev),
              seq=seq, pos=pos)
    if own:
        import synapse_b200 as sb
        ctx = sb.Context(torch.cuda.current_device())
        cache = sb.KVCache(ctx, top, c["kv"], c["hd"], 1, c["seqs"], c["page"], pt.next)
        for i in range(c["seqs"]):
            cache.advance(held[i], i)
        pools = cache.pages(0)
        pools[0].copy_(kp)
        pools[1].copy_(vp)
        st.update(ctx=ctx, cache=cache, pools=pools, new=new,
                  q_out=torch.empty(sum(new), c["heads"] * c["hd"], device=dev))
    return st


def _prepare_select(c, seed):
    g, dev = _gen(seed), "cuda"
    n = c["groups"] * c["beams"]
    # a language model's logits: a bulk and a few tokens that stand out
    x = torch.randn(n, c["vocab"], generator=g, device=dev) * 2.0
    hot = torch.randint(0, c["vocab"], (n, 20), generator=g, device=dev)
    x.scatter_add_(1, hot, 6 + 3 * torch.randn(n, 20, generator=g, device=dev))
    scores = -5 - 4 * torch.rand(n, generator=g, device=dev)
    fin = torch.zeros(n, dtype=torch.uint8, device=dev)
    fin[torch.randperm(n, generator=g, device=dev)[:c["done"]]] = 1
    st = dict(c=c, x=x, scores=scores, fin=fin, eos=min(2, c["vocab"] - 1))
    if own:
        import synapse_b200 as sb
        st.update(ctx=sb.Context(torch.cuda.current_device()))
    return st


def _prepare_reorder(c, seed):
    g, dev = _gen(seed), "cuda"
    r = random.Random(seed)
    n, b, page = c["groups"] * c["beams"], c["beams"], c["page"]
    # the prompt's full pages are shared, each beam's last ones are its own
    shared = c["length"] // 2 // page * page
    pt = _Pages(page)
    for gi in range(c["groups"]):
        first = []
        pt.grow(first, shared)
        pt.rows.append(first)
        for _ in range(b - 1):
            pt.rows.append(pt.fork(first, shared))
    for i in range(n):
        pt.grow(pt.rows[i], c["length"])
    # parents: `keep` beams of each group live on, the others take one's place
    par = []
    for _ in range(c["groups"]):
        live = sorted(r.sample(range(b), c["keep"]))
        par += [i if i in live else r.choice(live) for i in range(b)]
    shape = (c["layers"], pt.next, page, c["kv"], c["hd"])
    kp = torch.randn(shape, generator=g, device=dev)
    vp = torch.randn(shape, generator=g, device=dev)
    st = dict(c=c, k=kp, v=vp, table=pt.table(dev).int(),
              parents=torch.tensor(par, dtype=torch.int32, device=dev))
    if own:
        import synapse_b200 as sb
        ctx = sb.Context(torch.cuda.current_device())
        cache = sb.KVCache(ctx, max(c["length"], page), c["kv"], c["hd"], c["layers"], n, page,
                           pt.next)
        for gi in range(c["groups"]):
            cache.advance(shared, gi * b)
            for j in range(1, b):
                cache.fork(gi * b, gi * b + j, shared)
        for i in range(n):
            cache.advance(c["length"] - shared, i)
        pools = [cache.pages(li) for li in range(c["layers"])]
        for li in range(c["layers"]):
            pools[li][0].copy_(kp[li])
            pools[li][1].copy_(vp[li])
        whole = cache.pages()
        st.update(ctx=ctx, cache=cache, pools=whole, dev_table=cache.device_table(),
                  seqs=list(range(n)))
    return st


def prepare(case, seed):
    return {"attention": _prepare_attention, "append": _prepare_append,
            "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _norm_rope(x, w, cos, sin):
    """x [rows, heads, hd] in 32 bits; cos / sin [rows, hd/2]."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _run_attention(st):
    c = st["c"]
    if own:
        import synapse_b200 as sb
        out = sb.attention_decode_shared(st["plan"], 0, st["qkv"], None, None, EPS, st["cos"],
                                         st["sin"], window=c["window"])
        return {"out": out, "k": st["pools"][0], "v": st["pools"][1]}
    n, kv, hd, page = st["qkv"].shape[0], c["kv"], c["hd"], c["page"]
    grp, heads = c["heads"] // c["kv"], c["heads"]
    q, k, v = st["qkv"].view(n, -1, hd).split([heads, kv, kv], 1)
    cos, sin = st["cos"][st["lens"]], st["sin"][st["lens"]]
    q, k = _norm_rope(q, None, cos, sin), _norm_rope(k, None, cos, sin)
    row = torch.arange(n, device=q.device)
    at = (st["table"][row, st["lens"] // page], st["lens"] % page)
    st["k"].index_put_(at, k)
    st["v"].index_put_(at, v)
    # the prefix once for each group
    ng, nr = c["groups"], c["rows"]
    ip = torch.arange(st["pmax"], device=q.device)
    slot = (st["table"][::nr][:, ip // page], ip % page)
    kp, vp = st["k"][slot], st["v"][slot]                     # [ng, pmax, kv, hd]
    qg = q.view(ng, nr, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(ng, kv, nr * grp, hd)
    sp = (qg @ kp.permute(0, 2, 3, 1)).view(ng, kv, nr, grp, -1).permute(0, 2, 1, 3, 4)
    low = st["lens"] + 1 - (c["window"] or 1 << 30)
    pre = st["pre"].repeat_interleave(nr)
    okp = (ip < pre[:, None]) & (ip >= low[:, None])
    # what is each row's own
    pos = pre[:, None] + torch.arange(st["smax"], device=q.device)
    oks = (pos <= st["lens"][:, None]) & (pos >= low[:, None])
    pos = torch.minimum(pos, st["lens"][:, None])
    slot = (st["table"][row[:, None], pos // page], pos % page)
    ks, vs = st["k"][slot], st["v"][slot]                     # [n, smax, kv, hd]
    ss = q.view(n, kv, grp, hd) @ ks.permute(0, 2, 3, 1)
    s = torch.cat([sp.reshape(n, kv, grp, -1), ss], -1) / math.sqrt(hd)
    s = s.masked_fill(~torch.cat([okp, oks], -1)[:, None, None], -math.inf)
    e = (s - s.amax(-1, keepdim=True)).exp()
    e = e / e.sum(-1, keepdim=True)
    ep, es = e.split([st["pmax"], st["smax"]], -1)
    ep = ep.reshape(ng, nr, kv, grp, -1).permute(0, 2, 1, 3, 4).reshape(ng, kv, nr * grp, -1)
    op = (ep @ vp.permute(0, 2, 1, 3)).view(ng, kv, nr, grp, hd).permute(0, 2, 1, 3, 4)
    out = op.reshape(n, kv, grp, hd) + es @ vs.permute(0, 2, 1, 3)
    return {"out": out.reshape(n, heads * hd), "k": st["k"], "v": st["v"]}


def _run_append(st):
    c = st["c"]
    if own:
        import synapse_b200 as sb
        q = sb.qk_norm_rope_kv_append_batch(st["cache"], 0, range(c["seqs"]), st["new"],
                                            st["qkv"], c["heads"], st["qn"], st["kn"], EPS,
                                            st["cos"], st["sin"], q_out=st["q_out"])
        return {"q": q, "k": st["pools"][0], "v": st["pools"][1]}
    n, hd, page = st["qkv"].shape[0], c["hd"], c["page"]
    q, k, v = st["qkv"].view(n, -1, hd).split([c["heads"], c["kv"], c["kv"]], 1)
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    at = (st["table"][st["seq"], st["pos"] // page], st["pos"] % page)
    st["k"].index_put_(at, _norm_rope(k, st["kn"], cos, sin))
    st["v"].index_put_(at, v)
    return {"q": _norm_rope(q, st["qn"], cos, sin).reshape(n, -1), "k": st["k"], "v": st["v"]}


def _run_select(st):
    c = st["c"]
    if own:
        import synapse_b200 as sb
        s, p, t, f = sb.beam_select(st["ctx"], st["x"], st["scores"], c["beams"], k=c["k"],
                                    finished=st["fin"], eos=st["eos"])
        return {"scores": s, "parents": p, "tokens": t, "finished": f}
    g, b, v, k = c["groups"], c["beams"], c["vocab"], c["k"]
    x = st["x"].double()  # the order of near candidates hangs on more than 32 bits
    top = x.amax(-1, keepdim=True)
    lp = x - (top + (x - top).exp().sum(-1, keepdim=True).log())
    only = torch.where(torch.arange(v, device=x.device) == st["eos"], 0.0, -math.inf).double()
    fin = st["fin"].bool()
    lp = torch.where(fin[:, None], only, lp) + st["scores"].double()[:, None]
    # ties go to the lowest index: all above the k-th value, the first of those equal to it,
    # in the order of their indices, then sorted by value with that order kept
    lp = lp.view(g, b * v)
    edge = lp.topk(k, -1).values[:, -1:]
    at = torch.arange(b * v, device=x.device)
    over = torch.where(lp > edge, at, b * v).topk(k, -1, largest=False).values
    same = torch.where(lp == edge, at, b * v).topk(k, -1, largest=False).values
    same = torch.where(at[:k] < k - (over < b * v).sum(-1, keepdim=True), same.sort(-1).values, b * v)
    idx = torch.cat([over, same], -1).sort(-1).values[:, :k]
    idx = idx.gather(1, lp.gather(1, idx).sort(dim=-1, descending=True, stable=True).indices)
    parents, tokens = (idx // v).int(), (idx % v).int()
    done = (tokens == st["eos"]) | fin.view(g, b).gather(1, parents.long())
    return {"scores": lp.gather(1, idx).float(), "parents": parents, "tokens": tokens,
            "finished": done.to(torch.uint8)}


def _run_reorder(st):
    c = st["c"]
    if own:
        st["cache"].reorder(st["seqs"], st["parents"], c["beams"])
        return {"k": st["pools"][0], "v": st["pools"][1], "table": st["dev_table"]}
    n, b, page = st["parents"].shape[0], c["beams"], c["page"]
    full, tail = c["length"] // page, c["length"] % page
    base = torch.arange(n, device=st["table"].device) // b * b
    src = base + st["parents"].long()
    old = st["table"]
    new = old[src]
    # the last, part-filled page stays a sequence's own: the beams that live on
    # keep theirs, the others get a copy in the page that they had
    if tail:
        new[:, full] = old[:, full]
        a, d = old[src, full].long(), old[:, full].long()
        st["k"][:, d, :tail] = st["k"][:, a, :tail]
        st["v"][:, d, :tail] = st["v"][:, a, :tail]
    old.copy_(new)
    return {"k": st["k"], "v": st["v"], "table": old}


def run(state):
    return {"attention": _run_attention, "append": _run_append, "select": _run_select,
            "reorder": _run_reorder}[state["c"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "attention":
        pre, suf = _lengths(c)
        n, kvd, win = len(suf), c["kv"] * c["hd"], c["window"] or 1 << 30
        lens = [pre[i // c["rows"]] + s for i, s in enumerate(suf)]
        # of each group's prefix, what the row that sees furthest back reads; then each row's own
        seen = sum(p - max(0, min(lens[g * c["rows"]:(g + 1) * c["rows"]]) + 1 - win)
                   for g, p in enumerate(pre)
                   if p > max(0, min(lens[g * c["rows"]:(g + 1) * c["rows"]]) + 1 - win))
        mine = sum(min(s, win - 1) for s in suf)
        io = n * (2 * c["heads"] * c["hd"] + 4 * kvd)
        return {"bytes": 4 * (2 * kvd * (seen + mine) + io + n * c["hd"]),
                "flops": 4 * c["heads"] * c["hd"] * sum(min(x + 1, win) for x in lens)}
    if c["op"] == "append":
        n = sum(_counts(c)[1])
        vals = n * (c["heads"] + 2 * c["kv"]) * c["hd"]
        return {"bytes": 4 * (2 * vals + n * c["hd"]), "flops": 6 * n * (c["heads"] + c["kv"]) * c["hd"]}
    if c["op"] == "select":
        n = c["groups"] * c["beams"] - c["done"]
        return {"bytes": 4 * n * c["vocab"] + 13 * c["groups"] * c["k"] + 5 * c["groups"] * c["beams"],
                "flops": 4 * n * c["vocab"]}
    n = c["groups"] * c["beams"]
    copies = c["groups"] * (c["beams"] - c["keep"]) * (c["length"] % c["page"])
    return {"bytes": 16 * copies * c["layers"] * c["kv"] * c["hd"] + 8 * n * (c["length"] // c["page"] + 1)
            + 4 * n, "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits, row by row
# ---------------------------------------------------------------------------
def _rotated(x, w, cos, sin):
    """x [heads, hd] at one position, in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(torch.mean(x ** 2, 1, keepdim=True) + EPS) * w.double()
    h = x.shape[1] // 2
    y = torch.empty_like(x)
    y[:, :h] = x[:, :h] * cos.double() - x[:, h:] * sin.double()
    y[:, h:] = x[:, h:] * cos.double() + x[:, :h] * sin.double()
    return y


def _exact_attention(c, st):
    n, hd, page = st["qkv"].shape[0], c["hd"], c["page"]
    k, v = st["k"].double(), st["v"].double()
    flat_k, flat_v = k.view(-1, c["kv"], hd), v.view(-1, c["kv"], hd)
    out = torch.empty(n, c["heads"], hd, dtype=torch.float64, device=k.device)
    lens, table = st["lens"].tolist(), st["table"]
    for r in range(n):
        x = st["qkv"][r].view(-1, hd)
        end, co, si = lens[r], st["cos"][lens[r]], st["sin"][lens[r]]
        begin = max(0, end + 1 - c["window"]) if c["window"] else 0
        p = torch.arange(begin, end + 1, device=k.device)
        slots = table[r][torch.div(p, page, rounding_mode="floor")] * page + p.remainder(page)
        flat_k[slots[-1]] = _rotated(x[c["heads"]:c["heads"] + c["kv"]], None, co, si)
        flat_v[slots[-1]] = x[c["heads"] + c["kv"]:].double()
        q = _rotated(x[:c["heads"]], None, co, si).view(c["kv"], -1, hd)
        w = torch.softmax(torch.einsum("hgd,lhd->hgl", q, flat_k[slots]) / hd ** 0.5, -1)
        out[r] = torch.einsum("hgl,lhd->hgd", w, flat_v[slots]).reshape(-1, hd)
    return {"out": out.view(n, -1), "k": k, "v": v}


def _exact_append(c, st):
    hd, page = c["hd"], c["page"]
    k, v = st["k"].double(), st["v"].double()
    x = st["qkv"].double().view(st["qkv"].shape[0], -1, hd)
    z = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]][:, None]

    def turn(y, w):
        if w is not None:
            y = y * w.double() / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
        y = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * z
        return torch.cat([y.real, y.imag], -1)
    slots = st["table"][st["seq"], torch.div(st["pos"], page, rounding_mode="floor")] * page \
        + st["pos"].remainder(page)
    k.view(-1, c["kv"], hd)[slots] = turn(x[:, c["heads"]:c["heads"] + c["kv"]], st["kn"])
    v.view(-1, c["kv"], hd)[slots] = x[:, c["heads"] + c["kv"]:]
    return {"q": turn(x[:, :c["heads"]], st["qn"]).reshape(x.shape[0], -1), "k": k, "v": v}


def _exact_select(c, st):
    b, vocab, k, eos = c["beams"], c["vocab"], c["k"], st["eos"]
    res = [[], [], [], []]
    for g in range(c["groups"]):
        cand = []
        for j in range(b):
            r = g * b + j
            s0 = float(st["scores"][r])
            if st["fin"][r]:
                cand.append((-s0, j * vocab + eos, True))
                continue
            lp = torch.log_softmax(st["x"][r].double(), 0).cpu().numpy()
            best = np.argpartition(-lp, min(k, vocab - 1))[:k] if k < vocab else np.arange(vocab)
            best = np.nonzero(lp >= lp[best].min())[0]
            cand += [(-(s0 + float(lp[i])), j * vocab + int(i), int(i) == eos) for i in best]
        cand = sorted(cand)[:k]
        if len(cand) < k:
            return None  # fewer than k candidates are possible
        for (s, i, d) in cand:
            res[0].append(-s)
            res[1].append(i // vocab)
            res[2].append(i % vocab)
            res[3].append(d)
    shape, dev = (c["groups"], k), st["x"].device
    return {"scores": torch.tensor(res[0], dtype=torch.float64, device=dev).view(shape),
            "parents": torch.tensor(res[1], dtype=torch.int32, device=dev).view(shape),
            "tokens": torch.tensor(res[2], dtype=torch.int32, device=dev).view(shape),
            "finished": torch.tensor(res[3], dtype=torch.uint8, device=dev).view(shape)}


def _exact_reorder(c, st):
    k, v, table = st["k"].double(), st["v"].double(), st["table"].clone()
    full, tail = divmod(c["length"], c["page"])
    for i, p in enumerate(st["parents"].tolist()):
        s = i - i % c["beams"] + p
        table[i, :full] = st["table"][s, :full]
        if tail and s != i:
            a, d = int(table[s, full]), int(table[i, full])
            k[:, d, :tail] = k[:, a, :tail]
            v[:, d, :tail] = v[:, a, :tail]
    return {"k": k, "v": v, "table": table}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    if case["op"] == "append":
        return _exact_append(case, st)
    if case["op"] == "select":
        return _exact_select(case, st)
    return _exact_reorder(case, st)
