"""Decode attention over shared cache pages (syn_cuda_attention_decode_shared)
against the definition in 64 bits, and against the framework's own decode
attention."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")

U = 2.0 ** -24


@pytest.fixture(autouse=True, params=["0", "1", "2", "3"], ids=["chosen", "rows", "behind", "beside"])
def layout(request, monkeypatch):
    """Each of the ways in which a plan lays out its work; by itself it takes the fastest."""
    monkeypatch.setenv("SYN_PLAN_LAYOUT", request.param)


def _rope(n, hd):
    f = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float().cuda(), a.sin().float().cuda()


def _rand(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def _turn(x, w, cos, sin, eps):
    x = x.double()
    hd = x.shape[-1]
    if w is not None:
        x = x * w.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = cos.double(), sin.double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class Batch:
    """Groups of sequences: group g's first one holds pre[g] positions, the others fork
    it, then each grows by its own number."""

    def __init__(self, ctx, kv, heads, hd, page, pre, own, layers=1, seed=0, scale=1.0, spare=0):
        n = sum(len(o) for o in own)
        self.lens = [p + s for p, o in zip(pre, own) for s in o]
        self.kv, self.heads, self.hd, self.page = kv, heads, hd, page
        top = max(max(self.lens) + 4, page)
        pages = sum((x + 4 + page - 1) // page for x in self.lens) + spare if page else 0
        self.cache = c = sb.KVCache(ctx, top, kv, hd, layers, n, page, pages)
        self.groups, row = [], 0
        for p, o in zip(pre, own):
            rows = list(range(row, row + len(o)))
            c.advance(p, row)
            for j in rows[1:]:
                if page:
                    c.fork(row, j)
                else:
                    c.advance(p, j)
            for j, s in zip(rows, o):
                c.advance(s, j)
            self.groups.append(rows)
            row += len(o)
        if page:
            for i, t in enumerate(c.pages()):
                t.copy_(_rand(t.shape, seed + 1 + i, scale))
        else:
            for layer in range(layers):
                for j in range(n):
                    for i, t in enumerate(c.view(layer, j)):
                        t.copy_(_rand(t.shape, seed + 1 + i + 10 * j, scale))
        self.qkv = _rand((n, (heads + 2 * kv) * hd), seed + 5, scale)
        self.cos, self.sin = _rope(top, hd)
        self.plan = sb.DecodePlan(c, heads)
        self.plan.set(self.groups)

    def kv_of(self, layer, seq, n):
        if not self.page:
            return tuple(t[:n].view(n, self.kv, self.hd) for t in self.cache.view(layer, seq))
        pos = torch.arange(n)
        slot = self.cache.device_table()[seq].cpu()[pos // self.page].long() * self.page + pos % self.page
        return tuple(t.reshape(-1, self.kv, self.hd)[slot] for t in self.cache.pages(layer))

    def check(self, window=0, qn=None, kn=None, layer=0, eps=1e-6, out=None, lens=None):
        """The kernel's rows against 64 bits. Scores carry an absolute error e_s: operands of
        22 bits or more (each product at most 3 * 2^-22 off, plus its sums' roundings, hd / 8 + 8
        steps of 2^-24), the rotation's and norm's rounding of q and k (hd / 2 + 16 steps), all
        relative to |q||k| <= sum |q_i||k_i|; a softmax moves by at most 2 e_s relative, its sums
        add their own roundings: n additions in chains of at most n / 64 + 64, and 2 ulp an exp."""
        n, heads, kv, hd = len(self.lens), self.heads, self.kv, self.hd
        got = sb.attention_decode_shared(self.plan, layer, self.qkv, qn, kn, eps, self.cos, self.sin,
                                         window=window) if out is None else out
        x = self.qkv.view(n, -1, hd)
        for r, ln in enumerate(self.lens if lens is None else lens):
            k, v = (t.double().clone() for t in self.kv_of(layer, r, ln + 1))
            k[ln] = _turn(x[r, heads:heads + kv], kn, self.cos[ln], self.sin[ln], eps)
            v[ln] = x[r, heads + kv:].double()
            q = _turn(x[r, :heads], qn, self.cos[ln], self.sin[ln], eps).view(kv, -1, hd)
            lo = max(0, ln + 1 - window) if window else 0
            k, v = k[lo:], v[lo:]
            s = torch.einsum("hgd,lhd->hgl", q, k) / hd ** 0.5
            mag = torch.einsum("hgd,lhd->hgl", q.abs(), k.abs()).amax(-1) / hd ** 0.5
            p = torch.softmax(s, -1)
            want = torch.einsum("hgl,lhd->hgd", p, v)
            es = mag * (12 + hd / 8 + 8 + (hd / 2 + 16 if qn is not None or kn is not None else 6)) * U
            rel = 2 * es + (len(k) / 64 + 64 + 8 + 12) * U
            tol = rel[..., None] * torch.einsum("hgl,lhd->hgd", p, v.abs()) + 1e-30
            err = (got[r].view(kv, -1, hd).double() - want).abs()
            assert torch.isfinite(got[r]).all()
            assert (err <= tol).all(), (r, float((err / tol).max()))
        return got


CASES = [
    # kv heads, heads, hd, page, prefixes, positions of each row's own
    (8, 16, 128, 16, [64], [[3, 0, 1, 20]]),
    (2, 8, 64, 32, [300], [[150, 7, 33, 0, 64, 65, 31, 32]]),
    (1, 8, 128, 16, [1000], [[5] * 20]),                       # 160 query rows: two tiles
    (2, 2, 64, 24, [1, 100, 777], [[0, 0], [10], [1, 2, 3]]),  # groups, one row alone
    (2, 6, 96, 5, [63, 64, 65], [[0, 9], [4, 4, 4], [70, 1]]),
    (1, 1, 32, 7, [6, 7, 8], [[0, 0], [0, 0], [0, 0]]),
    (2, 32, 64, 16, [130], [[2, 1, 0]]),                       # 16 heads a KV head
    (1, 5, 20, 8, [70], [[1, 2]]),
    (2, 8, 128, 128, [128, 127], [[0, 1], [3, 0]]),
    (1, 4, 128, 64, [5000], [[40, 0, 3]]),                     # several CTAs a job
    (3, 3, 64, 1, [9], [[1, 2, 3]]),
    (2, 4, 128, 0, [70, 3], [[4, 5], [0]]),                    # contiguous: nothing shared
    (1, 2, 64, 16, [0, 0], [[0, 5], [0]]),                     # empty sequences
    (1, 8, 128, 64, [5000], [[40, 0, 3]]),
    (2, 16, 64, 16, [200, 90, 333], [[3, 9, 0], [1, 1], [5] * 9]),  # few and many query rows
    (1, 16, 96, 32, [100], [[0] * 40]),                        # five tiles of query rows
    (1, 24, 32, 4, [37, 4], [[1, 2], [3, 4]]),                 # 24 heads a KV head
    (4, 4, 128, 16, [], [[]]) if False else (4, 4, 128, 16, [3000], [[1]]),  # one long row
]


@pytest.mark.parametrize("kv,heads,hd,page,pre,own", CASES)
def test_against_64_bits(ctx, kv, heads, hd, page, pre, own):
    b = Batch(ctx, kv, heads, hd, page, pre, own, seed=hd + page)
    for g, (p, rows) in enumerate(zip(pre, b.groups)):
        want = p // page * page if page and len(rows) > 1 else 0
        assert all(b.plan.prefix(r) >= want for r in rows)
    b.check()
    b.check()  # the same call again, nothing left behind


@pytest.mark.parametrize("kv,heads,hd,page,pre,own", CASES[:6])
@pytest.mark.parametrize("window", [1, 2, 40, 100, 100000])
def test_window(ctx, kv, heads, hd, page, pre, own, window):
    Batch(ctx, kv, heads, hd, page, pre, own, seed=window).check(window=window)


def test_norms_layers_and_other_stream(ctx):
    b = Batch(ctx, 2, 8, 128, 16, [200], [[3, 40, 0]], layers=3, seed=3)
    qn, kn = _rand((128,), 50), _rand((128,), 51)
    for layer in (2, 0):
        b.check(qn=qn, kn=kn, layer=layer, eps=1e-5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sb.attention_decode_shared(b.plan, 1, b.qkv, qn, None, 1e-5, b.cos, b.sin)
    side.synchronize()
    b.check(qn=qn, layer=1, eps=1e-5, out=got)


@pytest.mark.parametrize("scale", [1e-4, 30.0])
def test_small_and_large_values(ctx, scale):
    """Scores near zero, and a softmax that is all but a maximum; values of both sizes."""
    Batch(ctx, 1, 4, 64, 16, [500], [[3, 90]], seed=9, scale=scale).check()


def test_value_scales_differ_between_positions(ctx):
    """Rows of K and V of very different magnitude in one tile, zero rows among them."""
    b = Batch(ctx, 1, 4, 128, 16, [256], [[3, 9]], seed=19)
    k, v = b.cache.pages(0)
    f = 10.0 ** torch.linspace(-6, 1, k.shape[0] * 16, device="cuda").view(-1, 16, 1, 1)
    k *= f.flip(0)
    v *= f
    k[2] = 0
    v[5, 3] = 0
    b.check()


def test_infinite_and_nan_rows_stay_with_their_readers(ctx):
    """What is masked (outside the window, behind the sequence, in unused pages) may hold
    anything."""
    b = Batch(ctx, 2, 4, 64, 16, [96], [[5, 20]], seed=4, spare=3)
    k, v = b.cache.pages(0)
    used = torch.zeros(b.cache.n_pages * 16, dtype=torch.bool, device="cuda")
    table = b.cache.device_table().cpu()
    b.check(window=0)
    for r, ln in enumerate(b.lens):
        pos = torch.arange(max(0, ln + 1 - 50), ln + 1)
        used[(table[r][pos // 16].long() * 16 + pos % 16).cuda()] = True
    for t, bad in ((k, float("nan")), (v, float("inf"))):
        t.view(-1, 2, 64)[~used] = bad
    b.check(window=50)


def test_equals_the_row_by_row_kernel(ctx):
    """The same step through attention_decode (flash): reassociation apart, the same."""
    b = Batch(ctx, 8, 32, 64, 32, [700], [[9] * 6], seed=2)
    got = b.check()
    other = sb.attention_decode(b.cache, 0, b.qkv, 32, None, None, 1e-6, b.cos, b.sin, batch=6, flash=True)
    assert float((got - other).norm() / other.norm()) < 2e-6


def test_steps_of_growing_beams(ctx):
    """Attention, advance, reorder in turn; the plan holds over all steps."""
    b = Batch(ctx, 2, 4, 64, 16, [50], [[0, 0, 0, 0]], seed=8)
    rng = np.random.default_rng(1)
    for step in range(3):
        b.qkv = _rand(b.qkv.shape, 100 + step)
        b.check()
        for s in range(4):
            b.cache.advance(1, s)
        b.lens = [x + 1 for x in b.lens]
        b.cache.reorder([0, 1, 2, 3], torch.tensor(rng.integers(0, 4, 4), dtype=torch.int32, device="cuda"), 4)


def test_captured_and_replayed_with_another_set(ctx):
    b = Batch(ctx, 2, 8, 128, 16, [96, 33], [[3, 0], [1, 1, 2]], seed=6)
    b.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sb.attention_decode_shared(b.plan, 0, b.qkv, None, None, 1e-6, b.cos, b.sin)
    for s in range(5):
        b.cache.advance(1, s)
    b.lens = [x + 1 for x in b.lens]
    for s in range(5):  # pages for the replay's positions
        b.cache.advance(1, s)
        b.cache.truncate(b.lens[s], s)
    b.plan.set(b.groups)
    sb.attention_decode_shared(b.plan, 0, b.qkv, None, None, 1e-6, b.cos, b.sin)  # reserves
    b.qkv.copy_(_rand(b.qkv.shape, 77))
    graph.replay()
    torch.cuda.synchronize()
    b.check(out=out)
    # another batch of five rows in the same plan
    b.plan.set([[4, 3, 2], [1, 0]])
    order = [4, 3, 2, 1, 0]
    graph.replay()
    torch.cuda.synchronize()
    lens, qkv = list(b.lens), b.qkv
    want = torch.empty_like(out)
    want[order] = out
    b.qkv = torch.empty_like(qkv)
    b.qkv[order] = qkv
    b.lens = lens
    b.check(out=want)


def test_captured_and_replayed_with_longer_prefixes(ctx):
    """Of lengths for which a plan by itself would choose another layout, both ways."""
    b = Batch(ctx, 8, 16, 128, 16, [32, 3000], [[1, 5, 0, 3] * 2, [2, 0, 40, 7] * 2], seed=8)
    lens, qkv = list(b.lens), b.qkv
    for first in (0, 1):
        b.plan = sb.DecodePlan(b.cache, b.heads)
        buf = torch.empty_like(qkv[:8])
        b.plan.set([b.groups[first]])
        sb.attention_decode_shared(b.plan, 0, buf, None, None, 1e-6, b.cos, b.sin)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sb.attention_decode_shared(b.plan, 0, buf, None, None, 1e-6, b.cos, b.sin)
        got = torch.empty(16, 16 * 128, device="cuda")
        for g in (1 - first, first):
            b.plan.set([b.groups[g]])
            buf.copy_(qkv[b.groups[g]])
            sb.attention_decode_shared(b.plan, 0, buf, None, None, 1e-6, b.cos, b.sin)  # reserves
            out.zero_()
            graph.replay()
            got[b.groups[g]] = out
        torch.cuda.synchronize()
        b.check(out=got, lens=lens)


def test_two_plans_on_two_streams(ctx):
    b = Batch(ctx, 2, 8, 64, 16, [400, 401], [[3, 0, 5], [1, 1, 2]], seed=6)
    plans = [sb.DecodePlan(b.cache, 8) for _ in range(2)]
    plans[0].set([[0, 1, 2]])
    plans[1].set([[3, 4, 5]])
    want = b.check()
    streams = [torch.cuda.Stream() for _ in range(2)]
    parts = [b.qkv[:3].contiguous(), b.qkv[3:].contiguous()]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(sb.attention_decode_shared(plans[i], 0, parts[i], None, None, 1e-6, b.cos, b.sin))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, outs[i][0])
            assert float((o - want[3 * i:3 * i + 3]).norm() / want.norm()) < 2e-6


def test_refusals(ctx):
    b = Batch(ctx, 2, 4, 64, 16, [40], [[3, 0, 5]], seed=1)
    for groups in ([[0, 0]], [[0, 3]], [[0], []], [[-1]], [[0, 1], [1, 2]]):
        with pytest.raises(sb.SynapseError) as e:
            b.plan.set(groups)
        assert e.value.status == 2, groups
    b.check()

    def call(qkv=b.qkv, layer=0, cos=b.cos, window=0, out=None, qn=None):
        sb.attention_decode_shared(b.plan, layer, qkv, qn, None, 1e-6, cos, b.sin, window=window, out=out)
    for kw, status in (({"qkv": b.qkv[:2]}, 4), ({"qkv": b.qkv.double()}, 2), ({"qkv": b.qkv.cpu()}, 2),
                       ({"layer": 1}, 2), ({"layer": -1}, 2), ({"cos": b.cos[:4]}, 4), ({"window": -1}, 2),
                       ({"out": b.qkv}, 4), ({"qn": b.cos[0, :3].contiguous()}, 4),
                       ({"qkv": b.qkv[:, :-1]}, 5)):
        with pytest.raises(sb.SynapseError) as e:
            call(**kw)
        assert e.value.status == status, kw
    with pytest.raises(sb.SynapseError) as e:
        sb.DecodePlan(b.cache, 3)
    assert e.value.status == 4
    with pytest.raises(sb.SynapseError) as e:
        sb.DecodePlan(sb.KVCache(ctx, 8, 1, 132, 1), 1)
    assert e.value.status == 12
    b.cache.truncate(41, 0)  # the plan no longer describes the sequence
    with pytest.raises(sb.SynapseError) as e:
        call()
    assert e.value.status == 2
    b.plan.set(b.groups)
    b.lens[0] = 41
    b.check()
    b.cache.advance(b.cache.max_seq - b.lens[2], 2)
    with pytest.raises(sb.SynapseError) as e:  # full
        call()
    assert e.value.status == 2
    b.plan.set([])
    assert sb.attention_decode_shared(b.plan, 0, b.qkv[:0], None, None, 1e-6, b.cos, b.sin).shape == (0, 256)
    b.cache.close()
    for act in (lambda: b.plan.set([[0]]), call):
        with pytest.raises(sb.SynapseError) as e:
            act()
        assert e.value.status == 1
