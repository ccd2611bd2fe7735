"""The cache's operators and the scores on torch's streams: a call without a
stream runs on the current one (also inside a capture), a call on another
stream than the current one keeps its memory until it is done with it."""
import numpy as np
import pytest
import torch

from catseye_b200 import score
from test_gpu_kv import blocks, check_attention, fill, make, randn, runs_of

pytestmark = pytest.mark.gpu
WAIT = 40_000_000   # clock cycles: some 20 ms, far beyond what a call takes


@pytest.fixture(autouse=True)
def _clean(gpu):
    yield
    torch.cuda.synchronize()


def late(t, value):
    """t becomes value on the current stream, after what takes some 20 ms."""
    torch.cuda._sleep(WAIT)
    t.copy_(value)


def test_scores_run_on_the_current_stream():
    x, new = randn(20, 3333, seed=1), randn(20, 3333, seed=2)
    t = torch.arange(20, dtype=torch.int32, device="cuda")
    want = score.logprobs(new, t, 5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late(x, new)
        got = score.logprobs(x, t, 5)
        copies = [g.clone() for g in got]
    side.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, copies))


def test_the_cache_runs_on_the_current_stream():
    c = make([70, 70], 2, 64, layers=1)
    fill(c, [70, 70])
    k, v, q, out, kb, vb = (torch.zeros(3, h, 64, device="cuda") for h in (2, 2, 4, 4, 2, 2))
    new = [randn(*x.shape, seed=i + 3) for i, x in enumerate((k, v, q))]
    spare = [p for p in range(c.n_pages) if p not in set(c.table.flatten().tolist())]
    last = int(c.table[0, 1])
    run = [(0, 3, 0, 65)]
    runs = runs_of(run)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x, n in zip((k, v, q), new):
            late(x, n)
        c.append(0, k, v, runs, 3)
        c.attention(0, out, q, runs, 3, 68)
        c.read(0, kb, vb, runs, 3)
        c.copy_pages([last], spare[:1])
    side.synchronize()
    check_attention(c, 0, new[2], out, run, 2)
    assert np.array_equal(kb.double().cpu().numpy(), blocks(new[0].double().cpu().numpy()))
    assert np.array_equal(vb.double().cpu().numpy(), blocks(new[1].double().cpu().numpy()))
    assert torch.equal(c.pool[spare[0]], c.pool[last])


def test_captured_without_a_stream():
    """Inside a capture the calls are part of it."""
    c = make([70], 1, 64, layers=1)
    fill(c, [70])
    x, t = randn(4, 900, seed=1), torch.arange(4, dtype=torch.int32, device="cuda")
    q, out = randn(1, 2, 64, seed=2), torch.zeros(1, 2, 64, device="cuda")
    runs = runs_of([(0, 1, 0, 69)])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = score.logprobs(x, t, 3)
        c.attention(0, out, q, runs, 1, 70)
    x.copy_(randn(4, 900, seed=5))
    q.copy_(randn(1, 2, 64, seed=6))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, score.logprobs(x, t, 3)))
    check_attention(c, 0, q, out, [(0, 1, 0, 69)], 2)


def test_dropped_results_of_another_stream_keep_their_memory():
    """Results of a call on another stream that are dropped at once: tensors made next on this one are not written over."""
    x, t = randn(600, 2000, seed=1), torch.zeros(600, dtype=torch.int32, device="cuda")
    want = score.logprobs(x, t, 5)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(WAIT)
        lp = score.logprobs(x, t, 5, stream=side.cuda_stream)[0]
        mine = [torch.full((600, n), 7, dtype=d, device="cuda") for n in (1, 5, 5, 1) for d in (torch.int32, torch.float32)]
        torch.cuda.synchronize()
        assert all((m == 7).all() for m in mine)
        assert torch.equal(lp, want)


def test_dropped_arguments_of_another_stream_keep_their_memory():
    c = make([200], 1, 64, layers=1)
    fill(c, [200])
    q = randn(90, 4, 64, seed=2)
    out, runs = torch.zeros_like(q), runs_of([(0, 90, 0, 110)])
    x = randn(300, 2000, seed=1)
    want = score.logprobs(x, None, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(WAIT)
    tmp, tmp2 = q.clone(), x.clone()
    side.wait_stream(torch.cuda.current_stream())
    c.attention(0, out, tmp, runs, 90, 200, stream=side.cuda_stream)
    got = score.logprobs(tmp2, None, 4, stream=side.cuda_stream)
    del tmp, tmp2
    noise = [torch.full_like(q, 1e3), torch.full_like(x, 1e3)]
    torch.cuda.synchronize()
    check_attention(c, 0, q, out, [(0, 90, 0, 110)], 4)
    assert all(torch.equal(a, b) for a, b in zip(want[1:], got[1:])) and len(noise) == 2
