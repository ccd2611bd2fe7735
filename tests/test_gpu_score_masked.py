"""Scores of rows that are mostly masked (-inf): what a constrained decode asks for."""
import math

import numpy as np
import pytest
import torch

from catseye_b200 import score
from test_gpu_score import check, logits, some

pytestmark = pytest.mark.gpu


def masked(rows, vocab, keep, seed, dtype=torch.float32):
    """All but `keep` tokens of every row at -inf."""
    x = logits(rows, vocab, seed, dtype)
    at = torch.rand(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").topk(keep).indices
    out = torch.full_like(x, -math.inf)
    return out.scatter(1, at, x.gather(1, at)), at[:, 0].to(torch.int32).contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 20), (3, 33), (2, 5000), (600, 4100), (1, 128000), (400, 32000)])
@pytest.mark.parametrize("keep,k", [(1, 1), (1, 32), (5, 20), (20, 32), (19, 8)])
def test_few_tokens_left(dtype, rows, vocab, keep, k):
    x, t = masked(rows, vocab, keep, rows + vocab + keep, dtype)
    t[::2] = 7                                                         # most likely masked
    check(x, t, k)


@pytest.mark.parametrize("vocab", [40000, 128000])
def test_allowed_tokens_behind_the_first_values(vocab):
    """Allowed: a whole stretch far behind, single tokens at the ends, an equal value by the thousand behind a mask."""
    x = torch.full((6, vocab), -math.inf, device="cuda")
    g = logits(6, vocab, 3)
    x[0, 30000:] = g[0, 30000:]
    x[1, [0, vocab - 1]] = g[1, [0, vocab - 1]]
    x[2, vocab - 3:] = 2.0
    x[3, 20000:29000] = -1.0
    x[4, 9000:9010] = torch.finfo(torch.float32).min                   # finite all the same
    x[5, 5000:5040] = g[5, 5000:5040]
    x[5, 30000:] = 50 + g[5, 30000:].abs()
    for k in (1, 9, 32):
        check(x, some(6, vocab), k)
    got = score.logprobs(x, None, 32)
    torch.cuda.synchronize()
    assert got[2][1].tolist() == sorted([0, vocab - 1], key=lambda i: -x[1, i].item()) + list(range(1, 31))
    assert got[3][1, 2:].eq(-math.inf).all()


@pytest.mark.parametrize("rows,k", [(1, 32), (16, 20), (1500, 32)])
def test_masked_rows_take_about_as_long(rows, k):
    vocab = 128000 if rows < 100 else 32000
    plain = logits(rows, vocab, 1)
    few, _ = masked(rows, vocab, 40, 2)
    behind = plain.clone()
    behind[:, :vocab // 2] = -math.inf
    tail = torch.full_like(plain, -math.inf)
    tail[:, -50:] = plain[:, -50:]
    took = []
    for x in (plain, few, behind, tail):
        each = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(200_000)                                 # the host is ahead
            a.record()
            score.logprobs(x, None, k)
            b.record()
            torch.cuda.synchronize()
            each.append(a.elapsed_time(b) * 1e3)
        took.append(round(float(np.median(each)), 1))
    print(rows, k, "us: plain, 40 left, half masked, the last 50 left:", took)
    assert max(took[1:]) < 2.5 * took[0] + 10, took
