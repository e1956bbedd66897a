"""Beam search of a model (Model.generate_beam, syn_cuda_generate_beam): the batched operators
of the beam search in a run, as a model uses them. The oracle is a beam search on the host in
64 bits over logits that a second model, with a contiguous cache, gives for one hypothesis at a
time. INT8 logits do not depend on the batch or on the cache's layout (bit-exact); the block
formats' carry the relative error of 1e-3 of the framework's other tests.

Where the gap between the last candidate that is kept and the first that is dropped is within the
error, the device may keep the other: the oracle finds, before the device runs, the number of steps up to
which every such gap is larger, and the search is compared over so many steps. Whatever the gaps, each
hypothesis' score must be the sum of its own tokens' log-probabilities (forced decoding).
"""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu

sb = pytest.importorskip("synapse_b200")
from synapse_b200 import synth  # noqa: E402

U = 2.0 ** -24
MAX_SEQ = 96
PROMPTS = {5: [3, 5, 7, 9, 11], 33: list(range(40, 73)), 1: [17], 48: list(range(300, 348))}


def _weights(fmt, name):
    cfg = synth.lm_config(name)
    if fmt == "INT8_KN":
        return cfg, synth.gen_lm_weights(cfg, fmt, seed=91)
    return cfg, synth.gen_lm_weights(cfg, fmt, seed=91,
                                     dequant=lambda f, b, n: O.dequant(f.name, b, n)[1])


def _logp(x):
    x = x.astype(np.float64)
    m = x.max()
    return x - (m + np.log(np.exp(x - m).sum()))


class Plain:
    """Logits behind prompt + tokens, one hypothesis at a time; and the search."""

    def __init__(self, ctx, cfg, w, fmt, prompt, max_seq=MAX_SEQ):
        self.m = sb.Model(ctx, cfg, w, max_seq)
        self.n = len(prompt)
        _, self.first = self.m.forward_prefill(prompt)
        self.memo = {(): self.first}
        self.rel = 0.0 if fmt == "INT8_KN" else 1e-3

    def logits(self, toks):
        toks = tuple(int(t) for t in toks)
        if toks not in self.memo:
            self.m.truncate(self.n)
            for i, t in enumerate(toks):
                _, lg = self.m.forward_one([t])
                self.memo[toks[:i + 1]] = lg[0].copy()
        return self.memo[toks]

    def step_error(self, x, score):
        """Of one step: the logit's and the log-sum-exp's errors; 86 U of the kernel's sum of
        exponentials (a 2 ulp exponential of an argument rounded at up to 20 log2(e), eight-way sums),
        and the f32 rounding of the score."""
        return 2 * self.rel * float(np.abs(x).max()) + (86 + abs(score)) * U

    def search(self, beams, steps, eos=-1):
        """(tokens, scores, error bound, steps that the bound settles)."""
        hyp, err, settled, ok = [((), 0.0, False)], 0.0, 0, True
        for t in range(steps):
            cand, e = [], 0.0
            for toks, s, fin in hyp:
                if fin:
                    cand.append((s, toks + (eos,), True))
                    continue
                x = self.logits(toks)
                lp = _logp(x)
                e = max(e, self.step_error(x, s + np.sort(lp)[-beams - 1]))
                for v in np.argsort(-lp, kind="stable")[:beams + 1]:
                    cand.append((s + lp[v], toks + (int(v),), v == eos))
            err += e
            cand.sort(key=lambda c: -c[0])
            ok = ok and (len(cand) <= beams or cand[beams - 1][0] - cand[beams][0] > 2 * err)
            settled += ok
            hyp = [(c[1], c[0], c[2]) for c in cand[:beams]]
        return [h[0] for h in hyp], np.array([h[1] for h in hyp]), err, settled

    def close(self):
        self.m.close()


def _check(plain, toks, scores, beams, steps, eos=-1):
    assert toks.shape == (beams, steps) and scores.shape == (beams,)
    assert (np.diff(scores) <= 0).all()
    assert len({tuple(r) for r in toks.tolist()}) == beams
    for row, score in zip(toks.tolist(), scores):
        s, err = 0.0, 0.0
        plain.logits(row[:-1])  # (and of all that lead there)
        for t, v in enumerate(row):
            x = plain.logits(row[:t])
            lp = _logp(x)
            err += plain.step_error(x, s)
            s += lp[v]
            if v == eos:
                assert all(u == eos for u in row[t:])
                break
        assert abs(s - score) <= err, (s, score, err)


def _paged(ctx, cfg, w, batch, page=16, pages=64):
    return sb.Model(ctx, cfg, w, MAX_SEQ, max_batch=batch, kv_page=page, kv_pages=pages)


@pytest.mark.parametrize("fmt,name,prompt,beams,steps", [
    ("INT8_KN", "tiny", 5, 4, 14), ("INT8_KN", "tiny", 33, 3, 10),
    ("INT8_KN", "tiny-window", 33, 4, 8), ("INT8_KN", "tiny", 1, 2, 6),
    ("Q4_0", "tiny", 5, 4, 8), ("Q4_0", "tiny", 33, 4, 8), ("Q4_0", "tiny", 33, 7, 20),
    ("Q4_0", "tiny-hd64", 48, 3, 6), ("Q4_0", "tiny-window", 33, 5, 12),
    ("Q8_0", "tiny-hd64", 33, 16, 5), ("INT8_KN", "tiny-hd64", 48, 64, 3)])
def test_search_equals_plain_search(ctx, fmt, name, prompt, beams, steps):
    cfg, w = _weights(fmt, name)
    plain = Plain(ctx, cfg, w, fmt, PROMPTS[prompt])
    *_, settled = plain.search(beams, steps)
    m = _paged(ctx, cfg, w, beams, pages=6 + 5 * beams)
    free = m.kv_pages_free()
    for n in sorted({steps, settled} - {0}):
        toks, scores = m.generate_beam(PROMPTS[prompt], n, beams)
        _check(plain, toks, scores, beams, n)
        if n == settled:
            want, ws, err, _ = plain.search(beams, n)
            assert sorted(map(tuple, toks.tolist())) == sorted(want)
            assert np.abs(np.sort(scores) - np.sort(ws)).max() <= err
        for b in range(beams):
            assert m.seq_len(b) == len(PROMPTS[prompt]) + n - 1
            m.reset(b)
        assert m.kv_pages_free() == free
    if fmt == "INT8_KN":
        assert settled >= 1
    m.close()
    plain.close()


@pytest.mark.parametrize("fmt,name", [("INT8_KN", "tiny"), ("Q4_0", "tiny-hd64")])
def test_sequences_hold_the_hypotheses(ctx, fmt, name):
    """The contexts after a search are the hypotheses': the next step's logits say so; for INT8
    bit for bit. Then the sequences go on as any others, and a new search may follow."""
    cfg, w = _weights(fmt, name)
    prompt = PROMPTS[33]
    plain = Plain(ctx, cfg, w, fmt, prompt)
    m = _paged(ctx, cfg, w, 6)
    for seq, steps in ((0, 20), (2, 17), (2, 2), (1, 1)):
        toks, _ = m.generate_beam(prompt, steps, 4, seq=seq)
        slots = [seq + i for i in range(4)]
        assert [m.seq_len(s) for s in slots] == [32 + steps] * 4
        _, lg = m.decode_slots(slots[::-1], toks[::-1, -1], want_logits=True)
        for i in range(4):
            want = plain.logits(toks[3 - i].tolist())
            if fmt == "INT8_KN":
                assert np.array_equal(lg[i], want)
            else:
                assert np.abs(lg[i] - want).max() <= 1e-3 * np.abs(want).max()
        for s in slots:
            m.reset(s)
    m.close()
    plain.close()


@pytest.mark.parametrize("fmt", ["INT8_KN", "Q4_0"])
def test_one_beam_is_greedy(ctx, fmt):
    cfg, w = _weights(fmt, "tiny")
    prompt = PROMPTS[5]
    plain = Plain(ctx, cfg, w, fmt, prompt)
    want, _, _, settled = plain.search(1, 30)
    m = _paged(ctx, cfg, w, 1)
    toks, scores = m.generate_beam(prompt, 30, beams=1)
    _check(plain, toks, scores, 1, 30)
    assert settled >= 1
    assert tuple(toks[0, :settled].tolist()) == want[0][:settled]
    m.close()
    plain.close()


@pytest.mark.parametrize("beams", [1, 3])
def test_eos(ctx, beams):
    """A token of the greedy continuation as the end: hypotheses that reach it are filled up with it;
    a search whose beams have all ended stops, and gives the pages that it had reserved back."""
    cfg, w = _weights("INT8_KN", "tiny")
    prompt = PROMPTS[5]
    plain = Plain(ctx, cfg, w, "INT8_KN", prompt)
    greedy = plain.search(1, 8)[0][0]
    eos = greedy[3]
    *_, settled = plain.search(beams, 12, eos)
    want = plain.search(beams, settled, eos)[0]
    m = _paged(ctx, cfg, w, beams)
    toks, scores = m.generate_beam(prompt, settled, beams, eos=eos)
    assert sorted(map(tuple, toks.tolist())) == sorted(want)
    _check(plain, toks, scores, beams, settled, eos)
    for b in range(beams):
        m.reset(b)
    steps = MAX_SEQ - len(prompt) + 1
    toks, scores = m.generate_beam(prompt, steps, beams, eos=eos)
    _check(plain, toks, scores, beams, steps, eos)
    if (toks[:, -1] == eos).all() and beams == 1:
        assert m.seq_len(0) < len(prompt) + steps - 1
        assert m.kv_pages_free() == 64 - (m.seq_len(0) + 15) // 16
    m.close()
    plain.close()


def test_graphs_and_eager_steps_agree(ctx, monkeypatch):
    """Steps replayed from a graph, launched one by one, and a graph kept from a search with another
    prompt, other sequences and, in between, a wider step that moves the scratch buffers."""
    cfg, w = _weights("Q4_0", "tiny")
    m = _paged(ctx, cfg, w, 8)
    first = m.generate_beam(PROMPTS[33], 12, 3)
    for b in range(3):
        m.reset(b)
    m.generate_beam(PROMPTS[48], 20, 8)
    for b in range(8):
        m.reset(b)
    again = m.generate_beam(PROMPTS[33], 12, 3, seq=4)
    for b in range(4, 7):
        m.reset(b)
    monkeypatch.setenv("SYN_RUNNER_GRAPH", "0")
    eager = m.generate_beam(PROMPTS[33], 12, 3)
    for other in (again, eager):
        assert np.array_equal(first[0], other[0])
        assert np.array_equal(first[1], other[1])
    m.close()


def test_more_steps_than_a_plan_is_kept_for(ctx):
    """300 steps: the plan is made again on the way, with what the beams share by then."""
    cfg, w = _weights("Q4_0", "tiny-hd64")
    plain = Plain(ctx, cfg, w, "Q4_0", PROMPTS[33], 340)
    m = sb.Model(ctx, cfg, w, 340, max_batch=4, kv_page=16, kv_pages=2 + 4 * 20)
    toks, scores = m.generate_beam(PROMPTS[33], 300, 4)
    _check(plain, toks, scores, 4, 300)
    _, lg = m.decode_slots([0, 1, 2, 3], toks[:, -1], want_logits=True)
    for row, x in zip(toks.tolist(), lg):
        want = plain.logits(row)
        assert np.abs(x - want).max() <= 1e-3 * np.abs(want).max()
    m.close()
    plain.close()


def test_pool_exhausted(ctx):
    """4 beams x 20 steps behind 33 tokens of 16-token pages: 2 + 4 * 2 = 10 pages."""
    cfg, w = _weights("INT8_KN", "tiny")
    m = _paged(ctx, cfg, w, 4, pages=9)
    with pytest.raises(sb.SynapseError) as e:
        m.generate_beam(PROMPTS[33], 20, 4)
    assert e.value.status == 3  # out of memory
    assert m.kv_pages_free() == 9 and [m.seq_len(i) for i in range(4)] == [0] * 4
    small = m.generate_beam(PROMPTS[33], 20, 3)
    m.close()
    m = _paged(ctx, cfg, w, 4, pages=10)
    four, _ = m.generate_beam(PROMPTS[33], 20, 4)
    for i in range(4):
        m.reset(i)
    again = m.generate_beam(PROMPTS[33], 20, 3)
    assert four.shape == (4, 20) and np.array_equal(small[0], again[0])
    m.close()


def test_refusals(ctx):
    cfg, w = _weights("INT8_KN", "tiny")
    m = sb.Model(ctx, cfg, w, MAX_SEQ, max_batch=2)
    with pytest.raises(sb.SynapseError) as e:  # a contiguous cache
        m.generate_beam([1, 2], 4, 2)
    assert e.value.status == 12  # unsupported
    m.close()
    m = _paged(ctx, cfg, w, 66, pages=80)
    bad = [dict(prompt=[]), dict(steps=0), dict(beams=0), dict(seq=64, beams=3), dict(seq=66),
           dict(seq=-1), dict(eos=512), dict(steps=MAX_SEQ, prompt=[1, 2]),
           dict(prompt=[1] * (MAX_SEQ + 1)), dict(beams=65)]
    for kw in bad:
        args = dict(prompt=[1, 2], steps=4, beams=2) | kw
        with pytest.raises(sb.SynapseError):
            m.generate_beam(**args)
    assert m.kv_pages_free() == 80
    m.forward_prefill([4, 5], seq=1)
    with pytest.raises(sb.SynapseError):  # a sequence in use
        m.generate_beam([1, 2], 4, 2)
    assert m.seq_len(0) == 0 and m.seq_len(1) == 2
    toks, _ = m.generate_beam([1, 2], MAX_SEQ - 1, 2, seq=2)  # up to the last position
    assert m.seq_len(2) == MAX_SEQ and toks.shape == (2, MAX_SEQ - 1)
    m.close()
