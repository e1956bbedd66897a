"""Decode plans and their attention where they can go wrong: caches of several head dims in one
process, reorders that cross a plan's groups, replays after other sets, values that are not
finite."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_shared_attention import Batch, _rand, _turn, layout  # noqa: F401 (layout: autouse)

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")

U = 2.0 ** -24


def _attend(b, plan=None, rows=None, layer=0, window=0):
    """One call for the rows (sequences) of a plan; output rows in the order of `rows`."""
    qkv = b.qkv if rows is None else b.qkv[rows].contiguous()
    return sb.attention_decode_shared(plan or b.plan, layer, qkv, None, None, 1e-6, b.cos, b.sin, window=window)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


ASCENDING = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import synapse_b200 as sb
from test_gpu_shared_attention import Batch
ctx = sb.Context(0)
for hd in (20, 32, 36, 60, 72, 80, 96, 112, 124):
    Batch(ctx, 1, 2, hd, 16, [70], [[1, 2]], seed=hd).check()
print("ascending ok")
"""


def test_head_dims_in_ascending_order():
    """A process whose caches get wider heads one after another (a kernel's shared memory grows
    with the head dim): in a process of its own, since others may have come in another order."""
    tests = os.path.dirname(os.path.abspath(__file__))
    code = ASCENDING.format(root=os.path.dirname(tests), tests=tests)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and "ascending ok" in out.stdout, out.stdout + out.stderr


def _refused(call, status=2):
    with pytest.raises(sb.SynapseError) as e:
        call()
    assert e.value.status == status


def test_reorder_across_the_plans_groups(ctx):
    """Two groups of two, and a reorder of all four: the second group's context moves into the
    first one. The plan has to be set again, and then describes the new contexts."""
    b = Batch(ctx, 2, 4, 64, 16, [64, 64], [[3, 3], [3, 3]], seed=3)
    b.check()
    b.cache.reorder([0, 1, 2, 3], _ints(2, 1, 0, 3), 4)
    _refused(lambda: _attend(b))
    b.plan.set(b.groups)
    b.check()
    b.cache.reorder([0, 1], _ints(1, 0), 2)  # inside a group: the plan holds
    b.check()


def test_reorder_with_a_sequence_outside_the_plan(ctx):
    """A beam that has ended is left out of the plan, and still takes part in the reorder."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 80], [[19, 19, 19, 19], [3]], seed=5)
    b.plan.set([[0, 1, 2]])
    # sequence 3 holds the same prompt: the shared pages stay what they are
    b.cache.reorder([0, 1, 2, 3], _ints(3, 3, 0, 1), 4)
    b.check(out=_attend(b, rows=[0, 1, 2]), lens=b.lens[:3])
    # sequence 4 does not
    b.cache.reorder([0, 1, 2, 4], _ints(3, 1, 2, 0), 4)
    _refused(lambda: _attend(b, rows=[0, 1, 2]))
    b.plan.set([[0, 1, 2]])
    b.check(out=_attend(b, rows=[0, 1, 2]), lens=b.lens[:3])


def test_reorder_through_a_sequence_outside_the_plan(ctx):
    """Another prompt's context comes into a sequence behind the plan's back, and from there
    into a row of the plan."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 64], [[3, 3, 3], [3]], seed=6)
    b.plan.set([[0, 1]])
    b.cache.reorder([2, 3], _ints(1, 0), 2)
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])
    b.cache.reorder([0, 2], _ints(1, 0), 2)
    _refused(lambda: _attend(b, rows=[0, 1]))
    b.plan.set([[0, 1]])
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])


def test_reorder_after_a_family_member_was_used_anew(ctx):
    """A sequence that held the shared pages when the plan was set, and no longer does."""
    b = Batch(ctx, 1, 4, 64, 16, [64], [[3, 3, 3]], seed=7, spare=12)
    b.plan.set([[0, 1]])
    b.cache.reset(2)
    b.cache.advance(67, 2)
    b.cache.reorder([0, 2], _ints(1, 0), 2)
    _refused(lambda: _attend(b, rows=[0, 1]))
    b.plan.set([[0, 1]])
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])


def test_captured_reorder_across_the_plans_groups(ctx):
    """A captured reorder may run at any time after a set: what its sequences do not all hold
    is not taken as shared."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 64], [[3, 3], [3, 3]], seed=8)
    par = _ints(0, 1, 2, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.cache.reorder([0, 1, 2, 3], par, 4)
    _refused(lambda: _attend(b))
    b.plan.set(b.groups)
    for p in ([2, 1, 0, 3], [3, 3, 0, 1]):
        par.copy_(_ints(*p))
        graph.replay()
        torch.cuda.synchronize()
        b.check()


def test_a_plan_outlives_its_cache(ctx):
    b = Batch(ctx, 1, 2, 64, 16, [40], [[3, 0]], seed=9)
    b.cache.close()
    _refused(lambda: b.plan.set([[0]]), 1)
    b.plan.close()


def test_errors_of_replays_are_reported(ctx):
    """What a replay cannot do is kept in the plan's error word: a position behind max_seq, and
    one for which no page was reserved."""
    b = Batch(ctx, 1, 4, 64, 16, [40], [[7, 0]], seed=21)
    c = b.cache  # max_seq 51
    assert b.plan.get_error() == 0
    b.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _attend(b)
    graph.replay()
    torch.cuda.synchronize()
    b.check(out=out)
    assert b.plan.get_error() == 0
    c.advance(1, 0)  # 48 positions: the next one needs a page
    graph.replay()
    assert b.plan.get_error() == 2
    assert b.plan.get_error() == 0
    b.lens[0] = 48
    b.check()  # takes the page
    graph.replay()
    torch.cuda.synchronize()
    b.check(out=out)
    assert b.plan.get_error() == 0
    c.advance(3, 0)
    graph.replay()
    assert b.plan.get_error() == 2


def test_error_word_of_a_closed_plan(ctx):
    b = Batch(ctx, 1, 2, 64, 16, [40], [[3, 0]], seed=22)
    b.plan.close()
    with pytest.raises(sb.SynapseError) as e:
        b.plan.get_error()
    assert e.value.status == 1


SETS = [[[0, 1, 2, 3], [4, 5, 6, 7]], [[0, 1], [2, 3, 4, 5, 6, 7]], [[0, 1, 2, 3, 4, 5, 6, 7]],
        [[0], [1], [2], [3], [4], [5], [6], [7]], [[0, 1], [2, 3], [4, 5], [6, 7]],
        [[0], [1, 2, 3, 4, 5, 6], [7]]]


def _capture(b, groups):
    b.plan = sb.DecodePlan(b.cache, b.heads)
    b.plan.set(groups)
    _attend(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _attend(b)
    return graph, out


@pytest.mark.parametrize("heads,prefix", [(1, 200), (4, 500), (4, 30), (16, 500)])
@pytest.mark.parametrize("first", range(len(SETS)))
def test_replay_after_any_set_of_as_many_rows(ctx, heads, prefix, first):
    """Groups of other sizes, other numbers of groups, groups of few query rows and of many, and
    rows for themselves, in the graph of one set: what the launches do is read from the plan."""
    b = Batch(ctx, 1, heads, 64, 16, [prefix], [[5, 0, 40, 3, 17, 16, 1, 33]], seed=heads)
    graph, out = _capture(b, SETS[first])
    for later in SETS + [SETS[first]]:
        b.plan.set(later)
        b.qkv.copy_(_rand(b.qkv.shape, len(later) + first))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        b.check(out=out)
        b.check()  # an eager call of the same set
    assert b.plan.get_error() == 0


def test_two_graphs_of_one_plan(ctx):
    """Captured under different sets: each replays under the other's, and under a third."""
    b = Batch(ctx, 1, 4, 64, 16, [2000], [[5, 0, 40, 3, 17, 16, 1, 33]], seed=2)
    b.plan.set(SETS[0])
    _attend(b)
    graphs = []
    for groups in (SETS[2], SETS[0], SETS[1]):
        b.plan.set(groups)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _attend(b)))
        graphs[-1] = (graph, graphs[-1][1])
    for groups in SETS:
        b.plan.set(groups)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            b.check(out=out)


def test_replay_after_a_set_of_another_number_of_rows(ctx):
    """No rows are computed, none appended; the output says so, and the plan's error word."""
    b = Batch(ctx, 1, 8, 64, 16, [200], [[5, 0, 40, 3]], seed=4)
    graph, out = _capture(b, [[0, 1, 2, 3]])
    for groups in ([[0, 1, 2]], [[3]], []):
        b.plan.set(groups)
        before = [t.clone() for t in b.cache.pages()]
        graph.replay()
        torch.cuda.synchronize()
        assert out.isnan().all()
        assert b.plan.get_error() == 2
        assert all(torch.equal(x, y) for x, y in zip(before, b.cache.pages()))
    b.plan.set([[0, 1, 2, 3]])
    graph.replay()
    torch.cuda.synchronize()
    b.check(out=out)
    assert b.plan.get_error() == 0


def _plain(b, window=0):
    """The definition in 64 bits, each row over the positions that it sees: [rows, kv, G, hd]
    and the weights' bound on the f32 error of finite outputs."""
    want, tol = [], []
    heads, kv, hd = b.heads, b.kv, b.hd
    x = b.qkv.view(len(b.lens), -1, hd)
    for r, ln in enumerate(b.lens):
        k, v = (t.double().clone() for t in b.kv_of(0, r, ln + 1))
        k[ln] = _turn(x[r, heads:heads + kv], None, b.cos[ln], b.sin[ln], 1e-6)
        v[ln] = x[r, heads + kv:].double()
        q = _turn(x[r, :heads], None, b.cos[ln], b.sin[ln], 1e-6).view(kv, -1, hd)
        lo = max(0, ln + 1 - window) if window else 0
        k, v = k[lo:], v[lo:]
        # (element by element: a library product may take 0 * inf another way)
        s = (q[:, :, None] * k.transpose(0, 1)[:, None]).sum(-1) / hd ** 0.5
        p = torch.exp(s - s.amax(-1, keepdim=True))  # NaN and infinities go their way
        p = p / p.sum(-1, keepdim=True)
        want.append((p[..., None] * v.transpose(0, 1)[:, None]).sum(-2))
        fin = [t.nan_to_num(0.0, 0.0, 0.0) for t in (q, k, v, p)]
        mag = torch.einsum("hgd,lhd->hgl", fin[0].abs(), fin[1].abs()).amax(-1) / hd ** 0.5
        es = mag * (12 + hd / 8 + 8 + 6) * U
        rel = 2 * es + (len(k) / 64 + 64 + 8 + 12) * U
        tol.append(rel[..., None] * torch.einsum("hgl,lhd->hgd", fin[3], fin[2].abs()) + 1e-30)
    return torch.stack(want), torch.stack(tol)


def _check_as_plain(b, window=0):
    """NaN and infinities where the definition has them (tolerances of finite outputs as in
    Batch.check), twice."""
    want, tol = _plain(b, window)
    for _ in range(2):
        got = _attend(b, window=window).view(want.shape).double()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got[got.isinf()], want[want.isinf()])
        fine = want.isfinite()
        assert ((got - want).abs()[fine] <= tol[fine]).all()
    assert b.plan.get_error() == 0
    if b.hd in (64, 128):  # the row-by-row kernel's NaN are in the same places
        other = sb.attention_decode(b.cache, 0, b.qkv.clone(), b.heads, None, None, 1e-6, b.cos, b.sin,
                                    window=window, batch=len(b.lens), flash=True).view(want.shape)
        assert torch.equal(other.isnan(), want.isnan())


SHAPES = [(1, 2, 64, 16, [96], [[40, 20]]),          # few query rows
          (2, 16, 128, 16, [300], [[3, 70, 0, 33]]),  # a tensor-core prefix
          (1, 12, 96, 5, [130, 60], [[4, 4], [70, 1]])]


def _place(b, seq, pos):
    t = b.cache.device_table()[seq].cpu()
    return int(t[pos // b.page]) * b.page + pos % b.page


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_queries_give_their_own_rows_nan(ctx, shape, bad):
    b = Batch(ctx, *shape, seed=11)
    b.qkv.view(len(b.lens), -1, b.hd)[1, b.heads - 1] = bad  # one head of one row
    _check_as_plain(b)
    got = _attend(b).view(len(b.lens), b.kv, -1, b.hd)
    assert got[1, -1, -1].isnan().all() and got.isnan().sum() == b.hd


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("first,n", [(0, 1), (0, 96), (17, 3), (33, 32)])
def test_nan_keys(ctx, shape, first, n):
    """In the first tile, as whole tiles, in between: NaN for every row that sees them, not zero."""
    b = Batch(ctx, *shape, seed=12)
    k, _ = b.cache.pages(0)
    for pos in range(first, first + n):
        k.view(-1, b.kv, b.hd)[_place(b, 0, pos), 0] = float("nan")
    _check_as_plain(b)
    assert _attend(b).view(len(b.lens), b.kv, -1)[0, 0].isnan().all()


@pytest.mark.parametrize("shape", SHAPES)
def test_nan_in_a_rows_own_positions(ctx, shape):
    b = Batch(ctx, *shape, seed=13)
    r = max(range(len(b.lens)), key=lambda i: b.lens[i])
    k, v = (t.view(-1, b.kv, b.hd) for t in b.cache.pages(0))
    k[_place(b, r, b.lens[r] - 1), -1, 3] = float("nan")
    _check_as_plain(b)
    k[_place(b, r, b.lens[r] - 1), -1, 3] = 0.0
    v[_place(b, r, b.lens[r] - 1), -1, 3] = float("nan")
    _check_as_plain(b)


@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_values_stay_in_their_columns(ctx, shape):
    """An infinity in V reaches its own column; the other columns keep that row's finite
    elements. With both signs in one column: NaN."""
    b = Batch(ctx, *shape, seed=14)
    v = b.cache.pages(0)[1].view(-1, b.kv, b.hd)
    v[_place(b, 0, 20), 0, 5] = float("inf")
    v[_place(b, 0, 21), 0, 6] = float("-inf")
    v[_place(b, 0, 22), 0, 7] = float("inf")
    v[_place(b, 0, 50), 0, 7] = float("-inf")
    _check_as_plain(b)
    row = _attend(b).view(len(b.lens), b.kv, -1, b.hd)[0, 0, 0]
    assert row[5] == float("inf") and row[6] == -float("inf") and row[7].isnan()
    assert row.isfinite().sum() == b.hd - 3


@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_keys(ctx, shape):
    """A score of +inf makes its row NaN (inf - inf), one of -inf weighs nothing."""
    b = Batch(ctx, *shape, seed=15)
    k, _ = b.cache.pages(0)
    k.view(-1, b.kv, b.hd)[_place(b, 0, 2), 0, 1] = float("inf")
    _check_as_plain(b)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window", [20, 45, 64])
def test_what_one_row_sees_and_another_does_not(ctx, shape, window):
    """Rows of a group end at different positions, so their windows begin at different ones: bad
    rows of the cache reach those that see them and no others."""
    b = Batch(ctx, *shape, seed=16)
    lens = sorted(b.lens[i] for i in b.groups[0])
    k, v = (t.view(-1, b.kv, b.hd) for t in b.cache.pages(0))
    pos = max(0, lens[0] + 1 - window)  # the first that the shortest row sees
    if pos < b.plan.prefix(b.groups[0][0]):
        v[_place(b, b.groups[0][0], pos), 0, 2] = float("inf")
        _check_as_plain(b, window)
        k[_place(b, b.groups[0][0], pos), 0, 2] = float("nan")
    _check_as_plain(b, window)


def test_scores_that_overflow(ctx):
    """Finite rows whose products pass the largest float: infinite scores, as in f32."""
    b = Batch(ctx, 1, 2, 64, 16, [96], [[40, 20]], seed=17)
    b.qkv[:, :2 * 64] = 1e25
    k, _ = b.cache.pages(0)
    k.view(-1, 1, 64)[_place(b, 0, 0):_place(b, 0, 0) + 16] = -1e25
    got = _attend(b)
    one = sb.attention_decode(b.cache, 0, b.qkv.clone(), 2, None, None, 1e-6, b.cos, b.sin, batch=2, flash=True)
    assert torch.equal(got.isnan(), one.isnan())


def test_a_parted_plan_says_so_everywhere(ctx):
    """Not only the attention call, of rows or of none, but what it would say of its rows too."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 64], [[3, 3], [3, 3]], seed=31)
    assert b.plan.prefix(1) == 64
    b.cache.reorder([0, 1, 2, 3], _ints(2, 1, 0, 3), 4)
    _refused(lambda: b.plan.prefix(1))
    _refused(lambda: _attend(b))
    b.plan.set(b.groups)
    assert b.plan.prefix(1) == 0
    b.check()


def test_more_tiles_than_32_bits_count(ctx, monkeypatch):
    """512 rows behind 2^26 shared positions, each by itself: refused, and the plan with it."""
    monkeypatch.setenv("SYN_PLAN_LAYOUT", "1")
    n, page = 512, 1 << 16
    cache = sb.KVCache(ctx, (1 << 26) + page, 1, 4, 1, n, page, 1024 + n)
    cache.advance(1 << 26, 0)
    for s in range(1, n):
        cache.fork(0, s)
    plan = sb.DecodePlan(cache, 1)
    plan.set([[0]])
    _refused(lambda: plan.set([list(range(n))]), 12)
    cos = torch.ones(cache.max_seq, 2, device="cuda")
    _refused(lambda: sb.attention_decode_shared(plan, 0, torch.zeros(1, 12, device="cuda"), None, None, 1e-6, cos, cos))
    _refused(lambda: plan.prefix(0))
    plan.set([list(range(256))])
    assert plan.prefix(255) == 1 << 26
    cache.close()


def test_replay_after_a_group_was_parted(ctx):
    """A replay asks nobody: the plan itself says that its rows are not what they were."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 64], [[3, 3], [3, 3]], seed=41, spare=8)
    graph, out = _capture(b, b.groups)

    def void():
        graph.replay()
        torch.cuda.synchronize()
        assert out.isnan().all() and b.plan.get_error() == 2

    def right():
        graph.replay()
        torch.cuda.synchronize()
        b.check(out=out)
        assert b.plan.get_error() == 0
    right()
    b.cache.reorder([0, 1, 2, 3], _ints(2, 1, 0, 3), 4)
    void()
    b.plan.set(b.groups)  # shares nothing now
    right()
    b = Batch(ctx, 1, 4, 64, 16, [64], [[3, 3, 5]], seed=42, spare=8)
    graph, out = _capture(b, b.groups)
    b.cache.reorder([0, 1], _ints(1, 0), 2)  # inside the group
    right()
    b.cache.truncate(66, 2)  # of its own positions
    b.lens[2] = 66
    right()
    b.cache.truncate(50, 2)  # of the shared ones
    void()
    b.lens[2] = 50
    b.plan.set(b.groups)
    b.check()
    right()
    b.cache.reset(0)
    void()
    b.lens[0] = 0
    b.plan.set(b.groups)
    b.check()
    right()


def _captured_reorder(b, seqs):
    par = torch.arange(len(seqs), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.cache.reorder(seqs, par, len(seqs))
    return graph, par


def test_what_a_captured_reorder_depends_on_is_used_anew(ctx):
    """A reorder of holders is captured after the set; one of them, outside the plan, then gets another
    context, which a replay would bring to the plan's rows."""
    b = Batch(ctx, 1, 4, 64, 16, [64], [[3, 3, 3, 3]], seed=51, spare=12)
    b.plan.set([[0, 1]])
    # 3 reaches the rows through 2 only, and was captured first
    graphs = [_captured_reorder(b, s) for s in ([2, 3], [0, 2])]
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])
    b.cache.reset(3)
    b.cache.advance(67, 3)
    _refused(lambda: _attend(b, rows=[0, 1]))
    b.plan.set([[0, 1]])
    for graph, par in graphs:
        par.copy_(_ints(1, 0))
        graph.replay()
    torch.cuda.synchronize()
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])


def test_a_holder_that_a_captured_reorder_may_replace(ctx):
    """Captured before the set: a sequence that holds the shared pages may have another context by the time
    an ordinary reorder brings it into the group."""
    b = Batch(ctx, 1, 4, 64, 16, [64, 64], [[3, 3, 3], [3]], seed=52)
    graph, par = _captured_reorder(b, [2, 3])
    b.plan.set([[0, 1]])
    par.copy_(_ints(1, 0))
    graph.replay()
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])
    b.cache.reorder([0, 2], _ints(1, 0), 2)
    _refused(lambda: _attend(b, rows=[0, 1]))
    b.plan.set([[0, 1]])
    b.check(out=_attend(b, rows=[0, 1]), lens=b.lens[:2])
