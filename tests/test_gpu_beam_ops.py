"""Beam-search operators on the paged cache against plain 64-bit forms: the
batched append (syn_cuda_qk_norm_rope_kv_append_batch), shared pages
(syn_cuda_kvcache_fork), reordering (syn_cuda_kvcache_reorder) and the
selection over beams x vocabulary (syn_cuda_beam_select)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")

U = 2.0 ** -24  # half a step of f32, relative


def _rope(n, hd):
    f = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float().cuda(), a.sin().float().cuda()


def _rand(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def _turn(x, w, cos, sin, eps):
    """([rows, heads, hd] in 64 bits, bound on an f32 evaluation's error)."""
    x = x.double()
    hd = x.shape[-1]
    rounds = 3
    if w is not None:
        x = x * w.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        # the sum of squares in up to hd/2 steps and 5 of a warp, root and quotient, 3 products
        rounds += hd // 2 + 12
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    bound = rounds * U * torch.cat([a.abs() + b.abs()] * 2, -1)
    return y, bound


def _slots(cache, seq, pos):
    t = cache.device_table()[seq].cpu()
    return t[pos // cache.page].long() * cache.page + pos % cache.page


@pytest.mark.parametrize("kv,heads,hd,page,norm,held,new", [
    (8, 16, 128, 16, True, [0, 15, 16, 40], [1, 1, 1, 1]),
    (2, 14, 64, 5, False, [3, 0, 7], [4, 0, 11]),
    (1, 1, 32, 64, True, [63, 64], [2, 130]),
    (3, 3, 96, 24, True, [10, 5, 1], [0, 3, 20]),
    (2, 4, 20, 8, True, [7, 2], [3, 1]),
    (1, 2, 256, 16, True, [1], [33]),
    (1, 2, 264, 16, True, [1, 4], [3, 2]),
    (2, 4, 80, 0, False, [6, 0], [2, 5]),
    (1, 2, 32, 4, True, [i % 7 for i in range(300)], [1 + i % 2 for i in range(300)]),
])
def test_append_batch(ctx, kv, heads, hd, page, norm, held, new):
    n, top = len(held), max(max(h + t for h, t in zip(held, new)), page) + 3
    pages = sum((h + t + page - 1) // page for h, t in zip(held, new)) if page else 0
    cache = sb.KVCache(ctx, top, kv, hd, 2, n, page, pages)
    for i, h in enumerate(held):
        cache.advance(h, i)
    if page:
        for p in cache.pages():
            p.copy_(_rand(p.shape, 3))
    rows = sum(new)
    qkv = _rand((rows, (heads + 2 * kv) * hd), 7)
    qn, kn = (_rand((hd,), 8), _rand((hd,), 9)) if norm else (None, None)
    cos, sin = _rope(top, hd)
    before = [p.clone() for p in cache.pages()] if page else None
    q = sb.qk_norm_rope_kv_append_batch(cache, 1, range(n), new, qkv, heads, qn, kn, 1e-5, cos, sin)
    x = qkv.view(rows, -1, hd)
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(new))
    pos = torch.cat([torch.arange(h, h + t) for h, t in zip(held, new)])
    want, bound = _turn(x[:, :heads], qn, cos[pos], sin[pos], 1e-5)
    assert ((q.view(rows, heads, hd).double() - want).abs() <= bound).all()
    wk, bk = _turn(x[:, heads:heads + kv], kn, cos[pos], sin[pos], 1e-5)
    if page:
        slot = torch.cat([_slots(cache, int(s), p[None]) for s, p in zip(seq, pos)])
        k, v = (p.view(2, -1, kv, hd) for p in cache.pages())
        assert ((k[1, slot].double() - wk).abs() <= bk).all()
        assert torch.equal(v[1, slot], x[:, heads + kv:])
        keep = torch.ones(k.shape[1], dtype=torch.bool)
        keep[slot] = False
        for now, was in zip((k, v), before):
            was = was.view(2, -1, kv, hd)
            assert torch.equal(now[0], was[0]) and torch.equal(now[1, keep], was[1, keep])
    else:
        for i in range(n):
            k, v = cache.view(1, i)
            at = pos[seq == i]
            assert ((k[at].view(-1, kv, hd).double() - wk[seq == i]).abs() <= bk[seq == i]).all()
            assert torch.equal(v[at].view(-1, kv, hd), x[seq == i, heads + kv:])
    for i, h in enumerate(held):
        assert cache.length(i) == h


def test_append_batch_in_place_unaligned_and_other_stream(ctx):
    kv, heads, hd, rows = 2, 4, 64, 6
    cache = sb.KVCache(ctx, 40, kv, hd, 1, 2, 8, 10)
    cos, sin = _rope(40, hd)
    flat = _rand((rows * (heads + 2 * kv) * hd + 1,), 5)
    odd = flat[1:].view(rows, -1)  # rows that start on 4 bytes only
    even = odd.clone()
    q1 = sb.qk_norm_rope_kv_append_batch(cache, 0, [1, 0], [4, 2], odd, heads, None, None, 1e-6, cos, sin)
    k1 = cache.pages(0)[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q2 = sb.qk_norm_rope_kv_append_batch(cache, 0, [1, 0], [4, 2], even, heads, None, None, 1e-6, cos, sin)
    side.synchronize()
    assert torch.equal(q1, q2) and torch.equal(k1, cache.pages(0)[0])


def test_append_batch_refusals(ctx):
    cache = sb.KVCache(ctx, 16, 2, 32, 1, 2, 8, 3)
    cos, sin = _rope(16, 32)
    qkv = _rand((2, 8 * 32), 1)

    def call(seqs, new, x=qkv, heads=4, layer=0, c=cos, q_out=None):
        return sb.qk_norm_rope_kv_append_batch(cache, layer, seqs, new, x, heads, None, None, 1e-6, c, sin,
                                               q_out=q_out)
    for args, status in (((([0, 0]), [1, 1]), 2), (([0, 2], [1, 1]), 2), (([0, -1], [1, 1]), 2),
                         (([0], [1]), 4), (([0, 1], [1]), 4), (([0], [17], _rand((17, 256), 1)), 2),
                         (([0, 1], [1, 1], qkv[:, :255]), 5), (([0, 1], [1, 1], qkv.double()), 2),
                         (([0, 1], [1, 1], qkv.cpu()), 2), (([0, 1], [1, 1], qkv, 3), 4),
                         (([0, 1], [1, 1], qkv, 4, 1), 2), (([0, 1], [1, 1], qkv, 4, -1), 2),
                         (([0, 1], [1, 1], qkv, 4, 0, cos[:8]), 4),
                         (([0, 1], [1, 1], qkv, 4, 0, cos, qkv), 4)):
        with pytest.raises(sb.SynapseError) as e:
            call(*args)
        assert e.value.status == status, args
    with pytest.raises(sb.SynapseError) as e:  # three pages, four needed; none is taken
        call([0, 1], [16, 9], _rand((25, 256), 1))
    assert e.value.status == 3
    cache.reset(0)
    cache.reset(1)
    assert cache.pages_free() == 3
    assert call([], [], qkv[:0]).shape == (0, 128)


# ---------------------------------------------------------------------------
# shared pages and reordering
# ---------------------------------------------------------------------------
class _Mirror:
    """What every sequence has to hold: its positions' values."""

    def __init__(self, cache):
        self.c, self.ctxs, self.tick = cache, [[] for _ in range(cache.batch)], 0

    def grow(self, seq, n):
        for _ in range(n):
            self.tick += 1
            x = torch.full((1, self.c.n_kv * self.c.hd), float(self.tick)).cuda()
            for layer in range(self.c.layers):
                self.c.append(layer, x + 0.25 * layer, -x - 0.25 * layer, seq)
            self.c.advance(1, seq)
            self.ctxs[seq].append(float(self.tick))

    def check(self):
        torch.cuda.synchronize()
        table = self.c.device_table().cpu()
        k, v = self.c.pages()
        for seq, want in enumerate(self.ctxs):
            assert self.c.length(seq) == len(want)
            if not want:
                continue
            pos = torch.arange(len(want))
            slot = table[seq][pos // self.c.page].long() * self.c.page + pos % self.c.page
            for layer in range(self.c.layers):
                w = (torch.tensor(want) + 0.25 * layer)[:, None].cuda()
                got_k = k[layer].reshape(-1, self.c.n_kv * self.c.hd)[slot]
                got_v = v[layer].reshape(-1, self.c.n_kv * self.c.hd)[slot]
                assert torch.equal(got_k, w.expand_as(got_k)), (seq, layer)
                assert torch.equal(got_v, -w.expand_as(got_v)), (seq, layer)


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("prompt", [1, 4, 9])
def test_fork_shares_full_pages(ctx, page, prompt):
    cache = sb.KVCache(ctx, 40, 1, 8, 3, 4, page, 80)
    m = _Mirror(cache)
    m.grow(2, prompt)
    free = cache.pages_free()
    for dst in (0, 3):
        cache.fork(2, dst)
        m.ctxs[dst] = list(m.ctxs[2])
    assert free - cache.pages_free() == (2 if prompt % page else 0)
    m.check()
    for seq in (0, 2, 3, 0):
        m.grow(seq, 3)
    m.check()
    # the source goes, the others keep the pages
    cache.reset(2)
    m.ctxs[2] = []
    m.grow(2, 5)
    m.check()
    # truncated into the shared part, then grown: its own copy, the other's is left alone
    cut = max(0, prompt - 1)
    cache.truncate(cut, 0)
    del m.ctxs[0][cut:]
    m.grow(0, 4)
    m.check()
    for seq in range(4):
        cache.reset(seq)
    assert cache.pages_free() == 80


def test_fork_refusals(ctx):
    flat = sb.KVCache(ctx, 16, 1, 8, 1, 2)
    cache = sb.KVCache(ctx, 16, 1, 8, 1, 3, 4, 5)
    m = _Mirror(cache)
    m.grow(0, 6)
    m.grow(1, 9)
    for c, args, status in ((flat, (0, 1, 0), 12), (cache, (0, 0, 1), 2), (cache, (0, 1, 1), 2),
                            (cache, (0, 2, 7), 2), (cache, (0, 3, 1), 2), (cache, (-1, 2, 1), 2),
                            (cache, (0, 2, -1), 2), (cache, (0, 2, 6), 3)):
        with pytest.raises(sb.SynapseError) as e:
            c.fork(*args)
        assert e.value.status == status, args
    cache.fork(0, 2, 4)  # a full page needs none
    m.ctxs[2] = m.ctxs[0][:4]
    m.check()
    cache.reset(2)
    cache.fork(0, 2, 0)
    assert cache.length(2) == 0


@pytest.mark.parametrize("page,groups,beams,prompt", [(4, 1, 4, 6), (1, 2, 3, 2), (16, 3, 8, 20),
                                                      (5, 1, 2, 5), (8, 1, 13, 3)])
def test_reorder_random_steps(ctx, page, groups, beams, prompt):
    n = groups * beams
    cache = sb.KVCache(ctx, 64, 2, 4, 2, n, page, n * ((64 + page - 1) // page))
    m, rng = _Mirror(cache), np.random.default_rng(page * 100 + beams)
    seqs = rng.permutation(n)
    for g in range(groups):
        first = int(seqs[g * beams])
        m.grow(first, prompt + g)
        for j in range(1, beams):
            dst = int(seqs[g * beams + j])
            cache.fork(first, dst)
            m.ctxs[dst] = list(m.ctxs[first])
    for step in range(14):
        par = rng.integers(0, beams, n)
        if step % 5 == 3:  # a permutation: nothing has to be copied
            par = np.concatenate([rng.permutation(beams) for _ in range(groups)])
        cache.reorder(seqs, torch.tensor(par, dtype=torch.int32, device="cuda"), beams)
        old = [list(c) for c in m.ctxs]
        for i in range(n):
            m.ctxs[seqs[i]] = list(old[seqs[i - i % beams + par[i]]])
        m.check()
        if step == 6:  # a beam that is cut back grows on its own
            for i in range(n):
                cache.truncate(prompt - 1, int(seqs[i]))
                del m.ctxs[seqs[i]][prompt - 1:]
        for i in range(n):
            m.grow(int(seqs[i]), 1 + step % 2 * 2)
    m.check()
    for i in range(n):
        cache.reset(i)
    assert cache.pages_free() == cache.n_pages


def test_reorder_odd_parents_and_refusals(ctx):
    cache = sb.KVCache(ctx, 32, 1, 8, 1, 4, 4, 32)
    m = _Mirror(cache)
    for s in range(4):
        m.grow(s, 6)
    par = torch.tensor([3, -1, 4, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    cache.reorder([0, 1, 2, 3], par, 4)  # indices out of range keep their own
    m.ctxs[0] = list(m.ctxs[3])
    m.check()
    ok = torch.zeros(4, dtype=torch.int32, device="cuda")
    flat = sb.KVCache(ctx, 16, 1, 8, 1, 4)
    for c, args, status in ((flat, ([0, 1], ok[:2], 2), 12), (cache, ([0, 0], ok[:2], 2), 2),
                            (cache, ([0, 4], ok[:2], 2), 2), (cache, ([0, 1, 2], ok[:3], 2), 4),
                            (cache, ([0, 1], ok, 2), 4), (cache, ([0, 1], ok[:2].long(), 2), 2),
                            (cache, ([0, 1], ok[:2].cpu(), 2), 2), (cache, ([0, 1], ok[:2], 0), 4)):
        with pytest.raises(sb.SynapseError) as e:
            c.reorder(*args)
        assert e.value.status == status, args
    m.grow(1, 1)
    with pytest.raises(sb.SynapseError):  # unequal lengths
        cache.reorder([0, 1], ok[:2], 2)
    cache.reorder([], ok[:0], 2)
    cache.reorder([1, 2], ok[:2], 1)
    m.check()


def test_reorder_captured_and_replayed(ctx):
    cache = sb.KVCache(ctx, 32, 1, 8, 2, 4, 4, 40)
    m = _Mirror(cache)
    m.grow(0, 6)
    for s in (1, 2, 3):
        cache.fork(0, s)
        m.ctxs[s] = list(m.ctxs[0])
    for s in range(4):
        m.grow(s, 1)
    par = torch.zeros(4, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder([0, 1, 2, 3], par, 4)
    m.check()
    for p in ([1, 0, 3, 3], [2, 2, 2, 1], [0, 1, 2, 3]):
        par.copy_(torch.tensor(p, dtype=torch.int32))
        graph.replay()
        old = [list(c) for c in m.ctxs]
        m.ctxs = [list(old[j]) for j in p]
        m.check()
    for s in range(4):  # the tables come back from the device
        cache.truncate(5, s)
        del m.ctxs[s][5:]
        m.grow(s, 5)
    m.check()
    for s in range(4):
        cache.reset(s)
    assert cache.pages_free() == 40


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
def _check_select(ctx, x, scores, beams, k, fin=None, eos=-1):
    """The result against the definition in 64 bits. Within a beam the order is exact
    (logit, then lower token). Between beams it is exact up to what the f32 sum of
    exponentials may be off, in halves of a step (U) relative to the sum: 2 ulp an exp, 4; its
    argument's rounding, at most |x - m| U with x - m <= 20 where it counts, 20; at most 3 + 16
    + 5 + 8 additions, 32; the factors that join threads and warps, twice (4 + 1 + at most 20 / 2
    on what is 20 / 2 below), 30. Two values differ by at most twice that."""
    tol = 86 * U
    n, vocab = x.shape
    got = sb.beam_select(ctx, x, scores, beams, k=k, finished=fin, eos=eos)
    s, p, t, f = (o.cpu().numpy() for o in got)
    big = np.finfo(np.float32).max
    xd = np.nan_to_num(x.cpu().numpy().astype(np.float64), nan=-np.inf, posinf=big, neginf=-np.inf)
    sd = np.nan_to_num(scores.cpu().numpy().astype(np.float64), nan=-np.inf, posinf=big, neginf=-np.inf)
    done = np.zeros(n, bool) if fin is None else fin.cpu().numpy().astype(bool)
    for g in range(n // beams):
        val = np.empty((beams, vocab))
        for b in range(beams):
            r = g * beams + b
            if done[r]:
                lp = np.full(vocab, -np.inf)
                lp[eos] = 0.0
            else:
                m = xd[r].max()
                with np.errstate(invalid="ignore"):
                    lp = xd[r] - (m + np.log(np.exp(xd[r] - m).sum())) if m > -np.inf else xd[r]
            val[b] = lp + sd[r]
        order = np.sort(val.reshape(-1))[::-1][:k]
        mine = val[p[g], t[g]]
        assert len({(a, b) for a, b in zip(p[g], t[g])}) == k
        fine = np.isfinite(order)
        assert np.array_equal(fine, np.isfinite(mine))
        assert (np.abs(mine[fine] - order[fine]) <= 2 * tol).all()
        assert (np.abs(s[g][fine] - order[fine]) <= 2 * tol + U * np.abs(order[fine])).all()
        assert np.isneginf(s[g][~fine]).all()
        for b in range(beams):  # each beam's first ones, in order
            took = t[g][p[g] == b]
            by = val[b] if done[g * beams + b] else xd[g * beams + b]
            ranked = np.argsort(-by, kind="stable")[:len(took)]
            assert np.array_equal(took[np.isfinite(val[b][took])], ranked[np.isfinite(val[b][ranked])])
        if not fine.all():  # equal values, -inf: by beam, then logit, then token
            flat = p[g].astype(np.int64)[~fine] * vocab + t[g][~fine]
            rest = np.nonzero(np.isneginf(val.reshape(-1)))[0]
            rows = g * beams + rest // vocab
            by = np.where(done[rows], 0.0, xd[rows, rest % vocab])
            rest = rest[np.lexsort((rest, -by, rest // vocab))][:len(flat)]
            assert np.array_equal(flat, rest)
        assert np.array_equal(f[g] != 0, done[g * beams + p[g]] | (t[g] == eos))
    return got


@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 3, 2, 6), (2, 4, 31, 4), (1, 5, 1000, 10), (3, 2, 8192, 4), (2, 3, 8193, 7),
    (1, 8, 151936, 16), (1, 64, 40000, 64), (40, 4, 32000, 8), (1, 2, 100001, 64), (9, 16, 16385, 32),
])
def test_select_random(ctx, groups, beams, vocab, k):
    n = groups * beams
    x = _rand((n, vocab), vocab + k, 3.0)
    scores = _rand((n,), 11, 2.0) - 5
    _check_select(ctx, x, scores, beams, k)
    _check_select(ctx, x, scores, beams, k, (torch.arange(n, device="cuda") % 3 == 1).to(torch.uint8),
                  vocab // 2)


@pytest.mark.parametrize("beams,vocab,k", [(4, 3000, 16), (1, 20000, 64), (64, 40001, 64)])
@pytest.mark.parametrize("kind", ["few", "same", "up", "down", "blocks", "zeros"])
def test_select_ties_and_shapes(ctx, beams, vocab, k, kind):
    i = torch.arange(vocab, device="cuda")
    x = {"few": (i * 7919 % 13).float(), "same": torch.full((vocab,), 2.5, device="cuda"),
         "up": i.float() / 64, "down": -i.float() / 64,
         # the best in the places of one thread of a segment
         "blocks": ((i // 4) % 256 == 17).float() * 10 + (i % 4) / 8,
         "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[kind]
    x = x.expand(beams, vocab).contiguous()
    scores = torch.zeros(beams, device="cuda")
    got = _check_select(ctx, x, scores, beams, k)
    # equal rows: the same sum, so equal values everywhere, and the lowest beam first
    flat = np.argsort(-np.tile(x[0].cpu().numpy().astype(np.float64), beams), kind="stable")[:k]
    assert np.array_equal(got[1].cpu().numpy()[0], flat // vocab)
    assert np.array_equal(got[2].cpu().numpy()[0], flat % vocab)


def test_select_infinities_nan_and_empty_rows(ctx):
    inf, nan = float("inf"), float("nan")
    x = _rand((8, 700), 3, 2.0)
    x[0] = -inf
    x[1] = nan
    x[2, 5] = inf
    x[3, ::2] = nan
    x[4, 3:] = -inf
    scores = torch.tensor([-1.0, -2, -3, -4, -5, -inf, nan, -6]).cuda()
    for beams, k in ((1, 8), (2, 8), (8, 64), (4, 3)):
        _check_select(ctx, x, scores, beams, k)
    fin = torch.ones(8, dtype=torch.uint8, device="cuda")
    _check_select(ctx, x, scores, 4, 9, fin, 699)
    _check_select(ctx, x, scores, 4, 4, fin, 0)


def test_select_strided_in_place_and_graph(ctx):
    wide = _rand((6, 5003), 2, 3.0)
    x = wide[:, 1:4100]  # odd start and stride
    scores = _rand((6,), 3) - 4
    fin = torch.tensor([0, 1, 0, 0, 0, 1], dtype=torch.uint8, device="cuda")
    want = _check_select(ctx, x, scores, 3, 3, fin, 9)
    s, f = scores.clone(), fin.clone()
    par, tok = torch.empty(2, 6, dtype=torch.int32, device="cuda")
    import ctypes
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert sb.lib.syn_cuda_beam_select(ctx.handle, p(x), 5003, 2, 3, 4099, p(s), p(f), 9, 3, p(s), p(par),
                                       p(tok), p(f), st) == 0
    for a, b in zip((s, par, tok, f), want):
        assert torch.equal(a.view(2, 3), b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sb.beam_select(ctx, x, scores, 3, finished=fin, eos=9)
    wide.copy_(_rand((6, 5003), 20, 3.0))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, _check_select(ctx, x, scores, 3, 3, fin, 9)):
        assert torch.equal(a, b)


def test_select_refusals(ctx):
    x, s = _rand((4, 50), 1), _rand((4,), 2)
    fin = torch.zeros(4, dtype=torch.uint8, device="cuda")
    for args, kw, status in (((x, s, 3), {}, 4), ((x, s, 0), {}, 4), ((x, s, 2), {"k": 0}, 4),
                             ((x, s, 2), {"k": 65}, 12), ((x[:, :1].contiguous(), s, 2), {"k": 3}, 2),
                             ((x, s[:3], 2), {}, 4), ((x.double(), s, 2), {}, 2), ((x.cpu(), s, 2), {}, 2),
                             ((x.t(), s, 2), {}, 5), ((x[:1].expand(4, 50), s, 2), {}, 5),
                             ((x, s, 2), {"finished": fin}, 2), ((x, s, 2), {"finished": fin, "eos": 50}, 2),
                             ((x, s, 2), {"finished": fin[:2], "eos": 1}, 4),
                             ((x, s, 2), {"finished": fin.int(), "eos": 1}, 2)):
        with pytest.raises(sb.SynapseError) as e:
            sb.beam_select(ctx, *args, **kw)
        assert e.value.status == status, (kw, status)
    wide = _rand((65, 10), 1)
    with pytest.raises(sb.SynapseError) as e:
        sb.beam_select(ctx, wide, _rand((65,), 2), 65)
    assert e.value.status == 12
    assert sb.beam_select(ctx, x[:0], s[:0], 2)[0].shape == (0, 2)


def test_views_keep_the_cache(ctx):
    """A view of the pools outlives the last name of its cache, but not its close()."""
    import weakref
    cache = sb.KVCache(ctx, 16, 1, 8, 2, 2, 4, 6)
    seen = weakref.ref(cache)
    k, table = cache.pages(1)[0], cache.device_table()
    del cache
    assert seen() is not None
    k.fill_(3.0)
    assert float(k.sum()) == 3.0 * k.numel()
    row = k[2:3]
    del k, table
    assert seen() is not None and float(row.sum()) == 96.0
    del row
    assert seen() is None
