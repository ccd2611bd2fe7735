"""Log probabilities, entropy and top alternatives of rows of logits
(catseye_b200.score) against the definition in 64 bits.

Tolerances.  A term e^(x - m) is off by 2^-21 relative (the difference exact to
2^-24 of |x - m| <= 32 where the term counts, the exponential 2 steps), a
thread's sum of n / 256 terms and the joins by (n / 256 + 16) 2^-24: the
logarithm of the sum is off by the two together, as is the entropy's quotient,
relative to 1 + |H|; differences of logits add 2^-23 of their size.  Ids are
compared for equality."""
import math

import numpy as np
import pytest
import torch

from catseye_b200 import _lib, score

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(gpu):
    gpu.cats_gpu_clear_device_error()
    yield


def reference(x, targets, k):
    x = x.double().cpu().numpy()
    m = x.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        e = np.exp(x - m)
        logs = np.log(e.sum(1, keepdims=True))
        lp = x - m - logs
        entropy = -np.where(e > 0, e * np.where(e > 0, lp, 0), 0).sum(1) / e.sum(1)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
    t = targets.cpu().numpy()
    got = np.where(t >= 0, lp[np.arange(len(x)), np.maximum(t, 0)], 0)
    return got, entropy, ids, np.take_along_axis(lp, ids, 1)


def check(x, targets, k, **kw):
    lp, h, ids, top = (a.cpu().numpy() for a in score.logprobs(x, targets, k, **kw))
    wlp, wh, wids, wtop = reference(x, targets, k)
    base = 2**-21 + (x.shape[1] / 256 + 16) * 2**-24
    fine = lambda a, w, extra=0: np.all((np.abs(a - w) <= base * (1 + extra) + 2**-22 * np.abs(w)) | (a == w))  # noqa: E731
    assert np.array_equal(ids[:, :wids.shape[1]], wids)
    assert fine(lp, wlp) and fine(top[:, :wtop.shape[1]], wtop)
    assert fine(h, wh, np.abs(wh))


def logits(rows, vocab, seed, dtype=torch.float32, scale=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype)


def some(rows, vocab, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (1, 31, 5), (5, 33, 32), (2, 1000, 0), (16, 32000, 5),
                                          (1, 32001, 20), (300, 4099, 8), (7, 131071, 32), (1, 256000, 1)])
def test_against_64_bits(dtype, rows, vocab, k):
    check(logits(rows, vocab, rows + vocab, dtype), some(rows, vocab), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 3), (5, 1)])
def test_rows_of_a_wider_tensor(dtype, pad, shift):
    wide = logits(9, 777 + pad, 3, dtype)
    wide[:, :shift] = math.nan
    wide[:, shift + 777 - max(pad - shift, 0) + pad:] = math.nan
    check(wide[:, shift:shift + 777 - shift], some(9, 700), 6)


def test_ties_go_to_the_lower_index():
    for vocab in (64, 5000, 32000):
        x = torch.zeros(4, vocab, device="cuda")
        x[1] = torch.arange(vocab, device="cuda") % 7                  # many equal maxima
        x[2, vocab - 1] = 1
        x[3] = -torch.arange(vocab, device="cuda").float() // 3
        check(x, some(4, vocab), 32)
    x = torch.full((1, 100), -0.0, device="cuda")
    x[0, 50:] = 0.0                                                     # -0 and 0 are equal
    assert score.logprobs(x, None, 32)[2][0].tolist() == list(range(32))


@pytest.mark.parametrize("vocab", [40, 3001, 70000])
def test_orders_that_keep_the_list_busy(vocab):
    x = torch.stack([torch.arange(vocab, device="cuda").float(), -torch.arange(vocab, device="cuda").float()]) * 1e-3
    check(x, some(2, vocab), 32)


@pytest.mark.parametrize("vocab", [37, 32000])
def test_masked_peaked_and_large_logits(vocab):
    x = logits(6, vocab, 1)
    x[0, 1:] = -math.inf                                                # one token left
    x[1, ::2] = -math.inf
    x[2] = -3e38
    x[3] *= 1e4                                                         # one token takes all
    x[4] += 1e4
    x[5, :] = torch.finfo(torch.float32).min
    x[5, 3] = 0
    t = some(6, vocab)
    t[0], t[1] = 2, 2                                                   # masked targets: -inf
    check(x, t, 4)
    lp, h, ids, top = score.logprobs(x, t, 4)
    assert lp[0] == -math.inf and h[0] == 0 and ids[0].tolist() == [0, 1, 2, 3] and top[0].tolist()[1:] == [-math.inf] * 3


def test_rows_without_a_distribution():
    x = logits(5, 3000, 1)
    x[0, 2999] = math.nan
    x[1, 5] = math.inf
    x[2] = -math.inf
    x[3, 7] = -math.inf
    lp, h, ids, top = score.logprobs(x, some(5, 3000), 3)
    assert lp[:3].isnan().all() and h[:3].isnan().all() and (ids[:3] == -1).all() and top[:3].isnan().all()
    assert lp[3:].isfinite().all() and (ids[3:] >= 0).all()


def test_targets_that_are_none_or_outside():
    x = logits(4, 100, 2)
    t = torch.tensor([-1, 5, 100, -100], dtype=torch.int32, device="cuda")
    lp = score.logprobs(x, t)[0]
    assert lp[0] == 0 and lp[3] == 0 and lp[2].isnan() and lp[1] < 0
    assert _lib.load().cats_gpu_device_error() == 0x20
    _lib.load().cats_gpu_clear_device_error()


def test_k_past_the_vocabulary_and_parts_not_wanted():
    x = logits(2, 5, 3)
    lp, h, ids, top = score.logprobs(x, None, 8, entropy=False)
    assert lp is None and h is None and (ids[:, 5:] == -1).all() and (top[:, 5:] == -math.inf).all()
    assert torch.equal(ids[:, :5].long(), torch.argsort(x, 1, descending=True))
    assert torch.allclose(top[:, :5].exp().sum(1), torch.ones(2, device="cuda"), atol=1e-6)
    assert score.logprobs(x[:0], some(0, 5), 2)[2].shape == (0, 2)


def test_captured_and_replayed():
    x, t = logits(20, 3333, 4), some(20, 3333)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        score.logprobs(x, t, 5, stream=s.cuda_stream)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            got = score.logprobs(x, t, 5, stream=s.cuda_stream)
    x.copy_(logits(20, 3333, 5))
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, score.logprobs(x, t, 5)):
        assert torch.equal(a, b)


def test_refusals():
    x, t = logits(3, 50, 1), some(3, 50)
    for f in (lambda: score.logprobs(x.cpu(), t), lambda: score.logprobs(x.double(), t), lambda: score.logprobs(x[0], t),
              lambda: score.logprobs(x, t.long()), lambda: score.logprobs(x, t[:2]), lambda: score.logprobs(x, t.cpu()),
              lambda: score.logprobs(x, t, 33), lambda: score.logprobs(x, t, -1), lambda: score.logprobs(x.t(), t),
              lambda: score.logprobs(x[:1].expand(3, 50), t)):
        with pytest.raises((ValueError, TypeError, _lib.CatsGpuError)):
            f()
