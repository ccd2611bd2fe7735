"""The batched step on the paged Q4_0 cache (cats_gpu_llm_cache_q4) and its
scores, against a float64 forward of the same weights that attends to the keys
and values the model's own cache holds, read back.

Tolerances.  Logits: the batched products' 2e-3 of the dense path
(test_gpu_batch.py, weights of 0.02), the probabilities' rounding to fp16,
2^-11, and what the rounding of the queries does to peaked attention, which
weights of 0.08 make: a normalised input times a matrix of N(0, w) gives
queries and keys of variance w^2 dim, so a score q k / sqrt(hs) carries
sqrt(sum (q_i k_i)^2) / sqrt(hs) = w^2 dim times the relative error of the
independent q_i.  That is 2^-11 / sqrt(3) rms from q's own rounding and 2^-11
from the product before it (fp16 weights and inputs, 2^-11 / sqrt(3) each, and
the same of the layer's input), together s = sqrt(4 / 3) 2^-11 w^2 dim.  A
probability p_j moves by p_j (s_j - mean), and the output sum p_j v_j by s of
its norm where the v_j are independent.  Two layers add in squares, and the
worst of some hundred rows lies three such deviations out: 3 sqrt(2) s.  The cache against the reference's keys and values:
a code is the nearest of 16 (half a step of the block's scale), save that the
value at minus the scale's side clamps to 7 of 8 steps (one step); a step is
an eighth of the block's largest magnitude, its scale rounded to 8 bits
(2^-9), and the product's 2e-3 comes on top."""
import numpy as np
import pytest

from models import ModelWeights, prompt, rel
from oracle.cpu import Q4_0, Q8_0

pytestmark = pytest.mark.gpu
W = 0.08


def tol(cfg):
    return 2e-3 + 2**-11 + 3 * 2**0.5 * (4 / 3)**0.5 * 2**-11 * W * W * cfg.dim


@pytest.fixture(scope="module")
def llm(gpu):
    from catseye_b200 import llm
    return llm


def config(llm, hs=32, mul=2, t=Q4_0, seq_len=320):
    heads = 2 * mul
    return llm.LlmConfig(dim=hs * heads, hidden=256, n_layers=2, n_heads=heads, n_kv_heads=2, vocab=512,
                         seq_len=seq_len, wtype=t)


def model(llm, orc, cfg, pages, seqs, cap=128, seed=5):
    # weights large enough that attention is far from uniform
    mw = ModelWeights(cfg, seed, orc, std=W)
    m = llm.GpuLLM(cfg)
    m.set_weights(mw)
    m.batch_reserve(cap, 1)
    m.cache_q4(pages, seqs)
    return mw, m


class Forward:
    """Logits of a sequence whose attention reads K/V rows given per layer."""

    def __init__(self, orc, mw):
        c = self.c = mw.cfg
        deq = lambda w, n, rows: orc.dequantize(c.wtype, w, n, rows).reshape(rows, n).astype(np.float64)  # noqa: E731
        per = lambda w, d, n: deq(w, n, c.n_layers * d).reshape(c.n_layers, d, n)                         # noqa: E731
        self.wq, self.wo = per(mw.wq, c.dim, c.dim), per(mw.wo, c.dim, c.dim)
        self.wk, self.wv = per(mw.wk, c.kv_dim, c.dim), per(mw.wv, c.kv_dim, c.dim)
        self.w1, self.w3 = per(mw.w1, c.hidden, c.dim), per(mw.w3, c.hidden, c.dim)
        self.w2, self.cls, self.emb = per(mw.w2, c.dim, c.hidden), deq(mw.wcls, c.dim, c.vocab), mw.emb.astype(np.float64)

    def rope(self, x, pos):
        n, d = x.shape
        hs = self.c.dim // self.c.n_heads
        i = np.arange(0, d, 2) % hs
        a = pos[:, None] / 10000.0 ** (i / hs)
        out = x.copy()
        out[:, 0::2] = x[:, 0::2] * np.cos(a) - x[:, 1::2] * np.sin(a)
        out[:, 1::2] = x[:, 0::2] * np.sin(a) + x[:, 1::2] * np.cos(a)
        return out

    def __call__(self, toks, cache):
        """cache(layer): K, V [n, kv_dim] the attention reads.  Returns logits and the K, V rows made on the way."""
        c, n = self.c, len(toks)
        hs, mul, pos = c.dim // c.n_heads, c.n_heads // c.n_kv_heads, np.arange(n)
        norm = lambda x: x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5)   # noqa: E731
        x, made = self.emb[toks], []
        for l in range(c.n_layers):
            h = norm(x)
            q = self.rope(h @ self.wq[l].T, pos)
            made.append((self.rope(h @ self.wk[l].T, pos), h @ self.wv[l].T))
            k, v = (a.astype(np.float64) for a in cache(l))
            att = np.zeros_like(x)
            for i in range(c.n_heads):
                kk, vv = (a[:, i // mul * hs:(i // mul + 1) * hs] for a in (k, v))
                s = q[:, i * hs:(i + 1) * hs] @ kk.T / np.sqrt(hs)
                s[np.triu_indices(n, 1)] = -np.inf
                p = np.exp(s - s.max(1, keepdims=True))
                att[:, i * hs:(i + 1) * hs] = p @ vv / p.sum(1, keepdims=True)
            x = x + att @ self.wo[l].T
            h = norm(x)
            g = h @ self.w1[l].T
            x = x + (g / (1 + np.exp(-g)) * (h @ self.w3[l].T)) @ self.w2[l].T
        return norm(x) @ self.cls.T, made


def check_cache(made, cache):
    for (k, v), (hk, hv) in zip(made, cache):
        for want, got in ((k, hk), (v, hv)):
            top = np.abs(want.reshape(-1, 32)).max(1, keepdims=True)
            step = top / 8 * (1 + 2**-8) + 2e-3 * np.abs(want).max()
            assert (np.abs(got.reshape(-1, 32) - want.reshape(-1, 32)) <= step).all()


@pytest.mark.parametrize("hs,mul", [(32, 2), (64, 1), (96, 2), (128, 2)])
@pytest.mark.parametrize("t", [Q4_0, Q8_0])
def test_ragged_prompts_and_single_tokens(llm, orc, hs, mul, t):
    """Three sequences of 70, 5 and 33 tokens in one call, their next tokens in
    a second, 40 more of the first in a third: logits and cache."""
    cfg = config(llm, hs, mul, t)
    mw, m = model(llm, orc, cfg, 12, 3)
    f = Forward(orc, mw)
    toks = [prompt(1, 111, cfg.vocab), prompt(2, 6, cfg.vocab), prompt(3, 34, cfg.vocab)]
    n0 = [70, 5, 33]
    got = [[], [], []]

    def call(parts):
        """parts: (sequence, from, to)"""
        nxt, lg = m.forward_batch(np.concatenate([toks[s][a:b] for s, a, b in parts]),
                                  np.concatenate([np.arange(a, b) for s, a, b in parts]),
                                  np.concatenate([np.full(b - a, s) for s, a, b in parts]), logits=True)
        assert (nxt == lg.argmax(1)).all()
        at = 0
        for s, a, b in parts:
            got[s].append(lg[at:at + b - a])
            at += b - a

    call([(s, 0, n0[s]) for s in (0, 1, 2)])
    call([(s, n0[s], n0[s] + 1) for s in (2, 0, 1)])
    call([(0, 71, 111)])
    for s in range(3):
        assert m.cache_length(s) == len(toks[s])
        held = [m.cache_read(l, s, len(toks[s])) for l in range(2)]
        want, made = f(toks[s], lambda l: held[l])
        check_cache(made, held)
        lg = np.concatenate(got[s])
        errs = [rel(lg[i], want[i]) for i in range(len(want))]
        assert max(errs) < tol(cfg), (s, max(errs))
    assert m.cache_free_pages == 12 - 2 - 1 - 1
    m.close()


def test_fork_truncate_compact(llm, orc):
    """A fork goes on as its source would and leaves it alone; truncated and
    compacted, the cache holds what it held."""
    cfg = config(llm, 64)
    _, m = model(llm, orc, cfg, 16, 4)
    toks = prompt(7, 150, cfg.vocab)
    m.forward_batch(toks[:100], np.arange(100), np.zeros(100, int))
    m.cache_fork(0, 1, 90)
    m.cache_fork(0, 2, 64)
    assert m.cache_free_pages == 14 and [m.cache_length(s) for s in range(4)] == [100, 90, 64, 0]
    before = [m.cache_read(l, 0, 100) for l in range(2)]
    # both write page 1: the source's positions 90.. and the fork's
    _, a = m.forward_batch(toks[90:130], np.arange(90, 130), np.full(40, 1), logits=True)
    for l in range(2):
        assert all(np.array_equal(x, y) for x, y in zip(before[l], m.cache_read(l, 0, 100)))
    _, b = m.forward_batch(toks[90:130], np.arange(90, 130), np.full(40, 0), logits=True)
    assert np.array_equal(a, b)
    _, c = m.forward_batch(toks[64:90], np.arange(64, 90), np.full(26, 2), logits=True)
    assert m.cache_free_pages == 16 - 3 - 2 - 1
    m.cache_truncate(0)
    with pytest.raises(RuntimeError):
        m.cache_read(0, 0, 1)
    keep = [m.cache_read(l, s, n) for l in range(2) for s, n in ((1, 130), (2, 90))]
    assert m.cache_compact() > 0
    again = [m.cache_read(l, s, n) for l in range(2) for s, n in ((1, 130), (2, 90))]
    assert all(np.array_equal(x[i], y[i]) for x, y in zip(keep, again) for i in (0, 1))
    _, d = m.forward_batch(toks[130:140], np.arange(130, 140), np.full(10, 1), logits=True)
    m.cache_fork(1, 3, 130)
    _, e = m.forward_batch(toks[130:140], np.arange(130, 140), np.full(10, 3), logits=True)
    assert np.array_equal(d, e)
    m.close()


def test_generation_from_forks(llm, orc):
    """Greedy decode of three sequences that share a prompt, across a page's
    end, in captured steps: every token is one its logits allow, and two
    sequences with the same context choose alike."""
    cfg = config(llm, 32)
    _, m = model(llm, orc, cfg, 16, 4)
    toks = prompt(8, 61, cfg.vocab)
    m.forward_batch(toks[:60], np.arange(60), np.zeros(60, int))
    for s in (1, 2):
        m.cache_fork(0, s, 60)
    start = np.array([toks[60], toks[60], 3], np.int32)
    out = m.generate_batch(start, [60, 60, 60], 10)
    assert np.array_equal(out[:, 0], out[:, 1])
    assert [m.cache_length(s) for s in range(3)] == [70] * 3
    seen = [m.cache_read(l, 2, 70) for l in range(2)]
    for s in (0, 2):
        m.cache_fork(s, 3, 60)
        fed = np.concatenate([[start[s]], out[:-1, s]])
        _, lg = m.forward_batch(fed, np.arange(60, 70), np.full(10, 3), logits=True)
        for i in range(10):
            assert lg[i, out[i, s]] >= lg[i].max() - 2 * tol(cfg) * np.linalg.norm(lg[i])
    for l in range(2):   # the captured steps wrote what a prompt's rows write, up to a step of the scale
        for x, y in zip(seen[l], m.cache_read(l, 3, 70)):
            assert np.array_equal(x[:60], y[:60])
            assert rel(x[60:], y[60:]) < 0.1
    # the same sequences again, from further on: the captured step is reused
    more = m.generate_batch(out[-1], [70, 70, 70], 5)
    assert np.array_equal(more[:, 0], more[:, 1])
    m.close()


def test_generation_planned_for_a_long_context(llm, orc):
    """A context long enough for the attention's other division of the work,
    captured; the first tokens of all are generated ones."""
    cfg = config(llm, 32, seq_len=32768)
    _, m = model(llm, orc, cfg, 16, 8)
    start = np.array([7, 7, 9, 9, 11, 13, 15, 7], np.int32)
    out = m.generate_batch(start, [0] * 8, 70)
    assert np.array_equal(out[:, 0], out[:, 1]) and np.array_equal(out[:, 0], out[:, 7]) and np.array_equal(out[:, 2], out[:, 3])
    for s in (0, 2, 6):
        fed = np.concatenate([[start[s]], out[:-1, s]])
        m.cache_truncate(s)
        _, lg = m.forward_batch(fed, np.arange(70), np.full(70, s), logits=True)
        for i in range(70):
            assert lg[i, out[i, s]] >= lg[i].max() - 2 * tol(cfg) * np.linalg.norm(lg[i])
    m.close()


def test_any_order_and_larger_batches(llm, orc):
    """Tokens of two sequences by turns, backwards, and a batch enlarged later:
    the logits of the grouped batch."""
    cfg = config(llm, 32)
    mw, m = model(llm, orc, cfg, 16, 4, cap=40)
    f = Forward(orc, mw)
    toks = [prompt(11, 100, cfg.vocab), prompt(12, 100, cfg.vocab)]
    pos = np.repeat(np.arange(20), 2)
    seqs = np.tile([0, 1], 20)
    order = np.concatenate([np.arange(0, 40, 3), np.arange(1, 40, 3)[::-1], np.arange(2, 40, 3)])
    mixed = np.array([toks[s][p] for s, p in zip(seqs, pos)])
    _, lg = m.forward_batch(mixed[order], pos[order], seqs[order], logits=True)
    m.batch_reserve(128, 1)
    assert m.cache_length(0) == 20
    _, more = m.forward_batch(np.concatenate([toks[0][20:], toks[1][20:44]]), np.concatenate([np.arange(20, 100), np.arange(20, 44)]),
                              np.repeat([0, 1], [80, 24]), logits=True)
    for s, n in ((0, 100), (1, 44)):
        held = [m.cache_read(l, s, n) for l in range(2)]
        want, made = f(toks[s][:n], lambda l: held[l])
        check_cache(made, held)
        got = {int(p): lg[i] for i, (p, q) in enumerate(zip(pos[order], seqs[order])) if q == s}
        got.update({20 + i: row for i, row in enumerate(more[:80] if s == 0 else more[80:])})
        assert max(rel(got[p], want[p]) for p in range(n)) < tol(cfg)
    m.close()


def test_enqueued_batches(llm, orc):
    """batch_set and its asynchronous steps: positions are made writable ahead
    of them, a batch is void once another call may have moved its pages, and
    steps past the context or the pool are refused."""
    cfg = config(llm, 32)
    _, m = model(llm, orc, cfg, 6, 3)
    start = np.array([5, 6], np.int32)
    want = m.generate_batch(start, [0, 0], 100)
    for s in (0, 1):
        m.cache_truncate(s)
    m.batch_set(start, [0, 0], [0, 1])
    m.batch_enqueue_decode(60)
    m.batch_enqueue_decode(40)
    m.batch_enqueue()                                 # the step at position 100, once more without moving on
    m.synchronize()
    assert [m.cache_length(s) for s in range(3)] == [101, 101, 0]
    _, a = m.forward_batch(want[-1], [100, 100], [0, 1], logits=True)
    m.cache_truncate(0, 100)
    m.cache_truncate(1, 100)
    _, b = m.forward_batch(want[-1], [100, 100], [0, 1], logits=True)
    assert np.array_equal(a, b)
    m.batch_set(want[-1], [100, 100], [0, 1])
    m.cache_fork(0, 2, 70)
    for call in (m.batch_enqueue, lambda: m.batch_enqueue_decode(1)):
        with pytest.raises(RuntimeError):
            call()
    kept = m.cache_read(0, 2, 70)
    m.batch_set(want[-1], [100, 100], [0, 1])
    with pytest.raises(RuntimeError):
        m.batch_enqueue_decode(300)
    m.batch_set(want[:5, 0], np.arange(101, 106), np.zeros(5, int))
    with pytest.raises(RuntimeError):                 # not one token a sequence
        m.batch_enqueue_decode(1)
    assert all(np.array_equal(x, y) for x, y in zip(kept, m.cache_read(0, 2, 70)))
    with pytest.raises(RuntimeError):
        m.cache_q4(2**31 - 1, 2)
    assert m.cache_length(2) == 70                    # refused: the cache as it was
    m.close()


def test_scores_and_dense_hand_over(llm, orc):
    """score_batch against the float64 softmax of the step's logits; the
    sequence copied into the single-token engine's cache goes on there."""
    cfg = config(llm, 64)
    mw, m = model(llm, orc, cfg, 8, 2)
    toks = prompt(9, 81, cfg.vocab)
    for paged in (True, False):
        if not paged:
            m.cache_q4(0)
        args = (toks[:80], np.arange(80))
        seqs = np.zeros(80, int)
        targets = toks[1:].copy()
        targets[5] = -1
        lp, h, ids, top = m.score_batch(*args, targets=targets, k=4, seqs=seqs)
        _, lg = m.forward_batch(*args, seqs, logits=True)
        z = lg.astype(np.float64)
        z = z - z.max(1, keepdims=True)
        z = z - np.log(np.exp(z).sum(1, keepdims=True))
        # a log probability: the argument's and the sum's roundings, and the answer's
        off = (np.abs(lg).max() + np.abs(z).max()) * 2**-22 + 2**-20
        hit = np.where(targets >= 0, z[np.arange(80), targets], 0)
        assert np.abs(lp - hit).max() <= off
        assert np.abs(h + (np.exp(z) * z).sum(1)).max() <= 8 * off
        assert np.array_equal(ids, np.argsort(-lg, axis=1, kind="stable")[:, :4])
        assert np.abs(top - np.take_along_axis(z, ids, 1)).max() <= off
        _, _, ids0, _ = m.score_batch(*args, seqs=seqs)
        assert ids0.shape == (80, 0)
        if paged:
            m.cache_to_dense(0, 80)
            got = m.step(int(toks[80]), 80)
            _, want = m.forward_batch(toks[80:], [80], [0], logits=True)
            # the engine quantizes its activations to Q8_0: each of 15 products
            # in a row is off by up to 2^-8 normwise
            assert rel(got, want[0]) < 15 * 2**-8
    m.close()


def test_refusals_leave_the_cache(llm, orc):
    cfg = config(llm, 32)
    _, m = model(llm, orc, cfg, 3, 2)
    toks = prompt(10, 100, cfg.vocab)
    m.forward_batch(toks[:70], np.arange(70), np.zeros(70, int))
    bad = [(toks[:2], [71, 72], [0, 0]),              # a gap
           (toks[:2], [5, 5], [0, 0]),                # a position twice
           (toks[:3], [10, 11, 10], [0, 0, 0]),
           (toks[:1], [0], [2]), (toks[:1], [0], [-1]),
           (toks[:1], [320], [0]), (toks[:2], [1, 2], [1, 1])]
    before = [m.cache_read(l, 0, 70) for l in range(2)]
    for t, p, s in bad:
        with pytest.raises(RuntimeError):
            m.forward_batch(t, p, s)
    with pytest.raises(RuntimeError):                 # three pages, two used
        m.forward_batch(toks[:65], np.arange(65), np.ones(65, int))
    with pytest.raises(RuntimeError):
        m.generate_batch(toks[:2], [70, 0], 80)
    for call in (lambda: m.cache_fork(0, 0, 10), lambda: m.cache_fork(0, 2, 10), lambda: m.cache_fork(0, 1, 71),
                 lambda: m.cache_truncate(0, 71), lambda: m.cache_truncate(2, 0), lambda: m.cache_read(2, 0, 1),
                 lambda: m.cache_read(0, 0, 71), lambda: m.cache_to_dense(1, 1), lambda: m.cache_q4(-1),
                 lambda: m.cache_q4(4, 0), lambda: m.score_batch(toks[:1], [70], targets=[512]),
                 lambda: m.score_batch(toks[:1], [70], k=33)):
        with pytest.raises(RuntimeError):
            call()
    assert m.cache_length(0) == 70 and m.cache_length(1) == 0 and m.cache_free_pages == 1
    for l in range(2):
        assert all(np.array_equal(x, y) for x, y in zip(before[l], m.cache_read(l, 0, 70)))
    m.cache_q4(0)
    assert m.cache_free_pages == -1 and m.cache_length(0) == -1
    for call in (lambda: m.cache_fork(0, 1, 0), lambda: m.cache_truncate(0, 0), m.cache_compact):
        with pytest.raises(RuntimeError):
            call()
    m.close()
    odd = llm.LlmConfig(dim=128, hidden=256, n_layers=1, n_heads=8, n_kv_heads=8, vocab=512, seq_len=64, wtype=Q4_0)
    n = llm.GpuLLM(odd)
    n.set_weights(ModelWeights(odd, 1, orc))
    with pytest.raises(RuntimeError):                 # heads of 16
        n.cache_q4(4, 1)
    n.close()
