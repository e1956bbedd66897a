"""The paged cache under captured calls, few pages and long searches; the selection's largest
sizes."""
import numpy as np
import pytest
import torch

from test_gpu_beam_ops import _Mirror, _check_select, _rand, _rope  # noqa: F401

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,prompt", [(4, 0), (4, 7), (5, 5), (1, 2)])
def test_captured_reorder_follows_the_lengths(ctx, page, prompt):
    """One graph for every step: the reorder's positions are those of the replay."""
    n = 4
    cache = sb.KVCache(ctx, 40, 1, 8, 2, n, page, n * 40)
    m, rng = _Mirror(cache), np.random.default_rng(page)
    if prompt:
        m.grow(0, prompt)
        for s in range(1, n):
            cache.fork(0, s)
            m.ctxs[s] = list(m.ctxs[0])
    par = _ints(0, 1, 2, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder(range(n), par, n)
    for step in range(12):
        for s in range(n):
            m.grow(s, 1 + step % 2)
        p = rng.integers(0, n, n)
        par.copy_(torch.tensor(p, dtype=torch.int32))
        graph.replay()
        old = [list(c) for c in m.ctxs]
        m.ctxs = [list(old[j]) for j in p]
        m.check()
    for s in range(n):
        cache.reset(s)
    assert cache.pages_free() == cache.n_pages


def test_captured_reorder_of_unequal_lengths(ctx):
    """A group whose lengths have parted by the replay stays as it is; the other one moves."""
    cache = sb.KVCache(ctx, 40, 1, 8, 1, 4, 4, 60)
    m = _Mirror(cache)
    for s in range(4):
        m.grow(s, 6)
    par = _ints(1, 0, 1, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder(range(4), par, 2)
    m.grow(1, 3)
    graph.replay()
    m.ctxs[2], m.ctxs[3] = m.ctxs[3], m.ctxs[2]
    m.check()


def test_cut_back_into_a_shared_page_before_a_replay(ctx):
    """A sequence that a graph may permute and that is cut back into a page which others hold
    gets its own copy at once: the replay writes there."""
    cache = sb.KVCache(ctx, 40, 1, 8, 2, 5, 4, 30)
    m = _Mirror(cache)
    for s in range(2):
        m.grow(s, 10)
    cache.fork(0, 4)  # holds sequence 0's full pages
    m.ctxs[4] = list(m.ctxs[0])
    par = _ints(0, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder([0, 1], par, 2)
    for s in range(2):
        cache.truncate(6, s)
        del m.ctxs[s][6:]
    par.copy_(_ints(1, 1))
    graph.replay()
    m.ctxs[0] = list(m.ctxs[1])
    m.check()  # (sequence 4 among them)
    for s in (0, 1, 4):
        m.grow(s, 5)
    m.check()
    for s in (0, 1, 4):
        cache.reset(s)
    assert cache.pages_free() == 30


def test_cut_back_without_a_page_for_the_copy(ctx):
    """Refused, and the sequence is as it was."""
    cache = sb.KVCache(ctx, 40, 1, 8, 1, 4, 4, 8)
    m = _Mirror(cache)
    m.grow(0, 8)
    cache.fork(0, 1)
    m.ctxs[1] = list(m.ctxs[0])
    par = _ints(0, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder([0, 1], par, 2)
    m.grow(2, 24)  # every other page
    assert cache.pages_free() == 0
    with pytest.raises(sb.SynapseError) as e:
        cache.truncate(6, 0)
    assert e.value.status == 3
    m.check()
    cache.truncate(20, 2)
    del m.ctxs[2][20:]
    cache.truncate(6, 0)
    del m.ctxs[0][6:]
    m.check()


def test_page_taken_while_capturing(ctx):
    """A captured append that takes a page, without a call before it: its replays find the page,
    and leave the table to the reorders in between."""
    kv, hd, page, n = 1, 8, 4, 4
    cache = sb.KVCache(ctx, 32, kv, hd, 1, n, page, 40)
    m = _Mirror(cache)
    m.grow(0, 8)  # full pages only
    for s in range(1, n):
        cache.fork(0, s)
        m.ctxs[s] = list(m.ctxs[0])
    cos, sin = _rope(32, hd)
    qkv = torch.zeros(n, 3 * hd, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sb.qk_norm_rope_kv_append_batch(cache, 0, range(n), [1] * n, qkv, 1, None, None, 1e-6, cos, sin)

    def step(value):
        qkv[:, 2 * hd:] = -torch.arange(n, device="cuda")[:, None] - value
        graph.replay()
        for s in range(n):
            cache.advance(1, s)
            m.ctxs[s].append(s + value)

    def check():  # V rows are stored as they come
        table, v = cache.device_table().cpu(), cache.pages(0)[1].reshape(-1, hd).cpu()
        for s, want in enumerate(m.ctxs):
            pos = torch.arange(len(want))
            got = v[table[s][pos // page].long() * page + pos % page]
            assert torch.equal(got, -torch.tensor(want)[:, None].expand_as(got)), s
    step(100.0)
    check()
    for value, p in ((200.0, [1, 0, 3, 2]), (300.0, [1, 2, 3, 0])):
        cache.reorder(range(n), _ints(*p), n)
        m.ctxs = [list(m.ctxs[j]) for j in p]
        check()
        step(value)
        check()


def test_page_taken_while_capturing_and_given_back(ctx):
    """A sequence that was cut back since has no page for the replay, which then writes nothing."""
    cache = sb.KVCache(ctx, 32, 1, 8, 1, 2, 4, 6)
    cos, sin = _rope(32, 8)
    qkv = torch.full((1, 24), 5.0, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sb.qk_norm_rope_kv_append_batch(cache, 0, [0], [1], qkv, 1, None, None, 1e-6, cos, sin)
    cache.reset(0)
    assert cache.pages_free() == 6
    for p in cache.pages():
        p.zero_()
    cache.advance(20, 1)  # all of the first one's pages, and more
    graph.replay()
    torch.cuda.synchronize()
    assert all(float(p.abs().sum()) == 0 for p in cache.pages())
    assert int((cache.device_table()[0] >= 0).sum()) == 0


def test_search_runs_in_the_pages_that_its_beams_hold(ctx):
    """Append, advance and reorder in turn, all beams from one: the pages of dropped beams are
    found again before a call is refused."""
    n, page, top = 4, 4, 64
    # the longest context once, and of each beam the page it writes and one before
    cache = sb.KVCache(ctx, top, 1, 8, 2, n, page, top // page + 2 * n)
    m = _Mirror(cache)
    m.grow(0, 16)
    for s in range(1, n):
        cache.fork(0, s)
        m.ctxs[s] = list(m.ctxs[0])
    for step in range(top - 16):
        for s in range(n):
            m.grow(s, 1)
        cache.reorder(range(n), _ints(*[step % n] * n), n)
        m.ctxs = [list(m.ctxs[step % n]) for _ in range(n)]
    m.check()
    for s in range(n):
        cache.reset(s)
    with pytest.raises(sb.SynapseError) as e:  # none left: refused, and nothing taken
        for s in range(n):
            cache.advance(top, s)
    assert e.value.status == 3
    for s in range(n):
        cache.reset(s)
    assert cache.pages_free() == cache.n_pages


def test_batched_calls_find_dropped_pages(ctx):
    """The same for the batched append and for a plan's attention."""
    n, page, hd = 4, 4, 8
    cos, sin = _rope(64, hd)
    for kind in ("append", "attention"):
        cache = sb.KVCache(ctx, 64, 1, hd, 1, n, page, 64 // page + 2 * n)
        cache.advance(16, 0)
        for s in range(1, n):
            cache.fork(0, s)
        plan = sb.DecodePlan(cache, 1)
        plan.set([list(range(n))])
        qkv = _rand((n, 3 * hd), 1)
        for step in range(64 - 17):
            if kind == "append":
                sb.qk_norm_rope_kv_append_batch(cache, 0, range(n), [1] * n, qkv, 1, None, None, 1e-6, cos, sin)
            else:
                sb.attention_decode_shared(plan, 0, qkv, None, None, 1e-6, cos, sin)
            for s in range(n):
                cache.advance(1, s)
            cache.reorder(range(n), _ints(*[step % n] * n), n)
        torch.cuda.synchronize()
        assert cache.length(0) == 63


def _grow(m, seq, n):
    """_Mirror.grow, with values that are made on the device (nothing waits for it)."""
    for _ in range(n):
        m.tick += 1
        for layer in range(m.c.layers):
            x = torch.full((1, m.c.n_kv * m.c.hd), m.tick + 0.25 * layer, device="cuda")
            m.c.append(layer, x, -x, seq)
        m.c.advance(1, seq)
        m.ctxs[seq].append(float(m.tick))


def test_growing_calls_after_a_captured_reorder_do_not_wait(ctx):
    """Sequences that a graph may permute at any time: appends, advances and attention find
    their pages on the device, with no wait for it."""
    n, hd, page = 4, 64, 4
    cache = sb.KVCache(ctx, 64, 1, hd, 2, n, page, 60)
    m = _Mirror(cache)
    m.grow(0, 9)
    for s in range(1, n):
        cache.fork(0, s)
        m.ctxs[s] = list(m.ctxs[0])
    par = _ints(0, 1, 2, 3)
    cos, sin = _rope(64, hd)
    plan = sb.DecodePlan(cache, 1)
    qkv = torch.zeros(n, 3 * hd, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder(range(n), par, n)
    plan.set([list(range(n))])
    # (every kernel once: a first launch loads it)
    sb.qk_norm_rope_kv_append_batch(cache, 0, range(n), [1] * n, qkv, 1, None, None, 1e-6, cos, sin)
    sb.attention_decode_shared(plan, 0, qkv, None, None, 1e-6, cos, sin)
    for s in range(n):
        _grow(m, s, 1)
    for p in ([1, 1, 3, 0], [2, 0, 1, 1]):
        par.copy_(torch.tensor(p, dtype=torch.int32))
        torch.cuda.synchronize()
        busy = torch.cuda.Event()
        torch.cuda._sleep(900_000_000)  # about half a second
        busy.record()
        graph.replay()
        m.ctxs = [list(m.ctxs[j]) for j in p]
        sb.qk_norm_rope_kv_append_batch(cache, 0, range(n), [1] * n, qkv, 1, None, None, 1e-6, cos, sin)
        sb.attention_decode_shared(plan, 1, qkv, None, None, 1e-6, cos, sin)
        for s in range(n):
            _grow(m, s, 3)  # (append and advance; over a page's end)
        assert not busy.query()
        m.check()
    for s in range(n):
        cache.reset(s)
    assert cache.pages_free() == 60


def test_captured_append_follows_a_reorder(ctx):
    """The rows of a replay go to the pages that its sequences have by then."""
    cache = sb.KVCache(ctx, 32, 1, 8, 2, 2, 4, 12)
    m = _Mirror(cache)
    for s in range(2):
        m.grow(s, 9)
    rows = torch.zeros(2, 3, 8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for s in range(2):
            for layer in range(2):
                cache.append(layer, rows[s], rows[s], s)
    cache.reorder([0, 1], _ints(1, 0), 2)
    m.ctxs.reverse()
    for s in range(2):
        rows[s] = 100.0 * (s + 1) + torch.arange(3, device="cuda")[:, None]
    graph.replay()
    torch.cuda.synchronize()
    m.check()
    table = cache.device_table().cpu()
    for s in range(2):
        pos = torch.arange(9, 12)
        slot = table[s][pos // 4].long() * 4 + pos % 4
        for t in cache.pages():
            for layer in range(2):
                assert torch.equal(t[layer].reshape(-1, 8)[slot], rows[s])


@pytest.mark.parametrize("vocab", [(1 << 24) + 3, 1 << 25])
def test_select_of_the_largest_vocabularies(ctx, vocab):
    """64 beams and 64 continuations: the header's limits, all at once."""
    beams = k = 64
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(beams, vocab, generator=g, device="cuda")
    x[torch.arange(beams), torch.randint(0, vocab, (beams,), generator=g, device="cuda")] = 9.0
    scores = -torch.rand(beams, generator=g, device="cuda")
    s, p, t, f = (o[0] for o in sb.beam_select(ctx, x, scores, beams, k=k))
    # each beam's k best logits in 64 bits; within a beam logits decide, and equal ones go to the
    # lower token
    val, tok, beam = [], [], []
    for b in range(beams):
        top, at = torch.topk(x[b], k + 8)
        lse = torch.logsumexp(x[b].double(), 0)
        val.append(scores[b].double() + (top.double() - lse))
        tok.append(at)
        beam.append(torch.full_like(at, b))
    val, tok, beam = torch.cat(val), torch.cat(tok), torch.cat(beam)
    best = val.sort(descending=True).values[:k]
    # as for smaller vocabularies: a thread's chain has an addition for every two tiles of its
    # segment, of which there are 800 at most, so ceil(16384 / 800 / 2) = 11 of the 16 counted there
    tol = 2 * 86 * 2.0 ** -24
    mine = scores[p.long()].double() + (x[p.long(), t.long()].double()
                                        - torch.stack([torch.logsumexp(x[b].double(), 0) for b in p.tolist()]))
    assert ((mine - best).abs() <= tol).all()
    assert ((s.double() - best).abs() <= tol + 2.0 ** -24 * best.abs()).all()
    assert len({(a, b) for a, b in zip(p.tolist(), t.tolist())}) == k
    for b in set(p.tolist()):
        took = x[b, t[p == b].long()]
        assert torch.equal(took, torch.topk(x[b], len(took)).values)


def test_select_end_tokens_that_are_no_int32(ctx):
    x, s, fin = _rand((2, 50), 1), _rand((2,), 2), torch.zeros(2, dtype=torch.uint8, device="cuda")
    for eos in (2 ** 32 + 9, 2 ** 31, -2 ** 31 - 1):
        with pytest.raises(sb.SynapseError) as e:
            sb.beam_select(ctx, x, s, 2, finished=fin, eos=eos)
        assert e.value.status == 2
    sb.beam_select(ctx, x, s, 2, finished=fin, eos=9)


def test_captured_select_outlives_a_larger_one():
    """The context's scratch grows between a capture and its replay: the graph's own stays."""
    ctx = sb.Context(0)
    x, s = _rand((4, 3000), 1, 3.0), _rand((4,), 2)
    want = [t.clone() for t in sb.beam_select(ctx, x, s, 4)]
    graphs = []
    for rows in (4, 4, 64, 512):
        big, bs = _rand((rows, 20000), rows, 3.0), _rand((rows,), 3)
        sb.beam_select(ctx, big, bs, 4)  # (grows from the third on)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sb.beam_select(ctx, x, s, 4)
        graphs.append((graph, out))
    fill = [torch.full((1 << 22,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]
    for graph, out in graphs + graphs:
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    assert all(int((t != 7).sum()) == 0 for t in fill)
    del graphs, graph
    ctx.close()
