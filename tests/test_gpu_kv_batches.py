"""The batched step on the paged Q4_0 cache: what its calls leave behind when
they do not run, run late or run out of room."""
import numpy as np
import pytest

from models import prompt
from test_gpu_kv_model import config, llm, model  # noqa: F401

pytestmark = pytest.mark.gpu


def start(llm, orc, pages=6, seqs=3, n=70, **kw):
    cfg = config(llm, 32, **kw)
    _, m = model(llm, orc, cfg, pages, seqs)
    toks = prompt(10, 200, cfg.vocab)
    m.forward_batch(toks[:n], np.arange(n), np.zeros(n, int))
    return m, toks


def test_no_steps_leave_no_position(llm, orc):
    m, toks = start(llm, orc)
    free = m.cache_free_pages
    assert m.generate_batch(toks[70:72], [70, 0], 0).shape == (0, 2)
    assert [m.cache_length(s) for s in range(3)] == [70, 0, 0] and m.cache_free_pages == free
    with pytest.raises(RuntimeError):
        m.cache_read(0, 0, 71)
    with pytest.raises(RuntimeError):                 # a gap, as ever
        m.generate_batch(toks[70:71], [71], 0)
    with pytest.raises(RuntimeError):
        m.forward_batch(toks[71:72], [71], [0])
    m.close()


def test_a_batch_that_never_ran_leaves_no_position(llm, orc):
    m, toks = start(llm, orc)
    _, want = m.forward_batch(toks[70:72], [70, 71], [0, 0], logits=True)
    m.cache_truncate(0, 70)
    m.batch_set(toks[70:72], [70, 71], [0, 0])
    assert m.cache_length(0) == 70
    with pytest.raises(RuntimeError):                 # 70 and 71 were not written
        m.forward_batch(toks[72:73], [72], [0])
    with pytest.raises(RuntimeError):
        m.cache_read(0, 0, 72)
    with pytest.raises(RuntimeError):
        m.cache_fork(0, 1, 72)
    m.batch_set(toks[70:72], [70, 71], [0, 0])
    m.batch_enqueue()
    m.synchronize()
    assert m.cache_length(0) == 72
    _, got = m.forward_batch(toks[70:72], [70, 71], [0, 0], logits=True)
    assert np.array_equal(got, want)
    m.close()


def test_pages_of_a_batch_that_never_ran_are_free_for_the_next(llm, orc):
    m, toks = start(llm, orc, pages=4)                # two pages left
    m.batch_set(toks[:128], np.arange(128), np.ones(128, int))
    m.batch_set(toks[:65], np.arange(65), np.full(65, 2))
    m.batch_enqueue()
    m.synchronize()
    assert [m.cache_length(s) for s in range(3)] == [70, 0, 65] and m.cache_free_pages == 0
    _, a = m.forward_batch(toks[65:68], np.arange(65, 68), np.full(3, 2), logits=True)
    _, b = m.forward_batch(toks[65:68], np.arange(65, 68), np.zeros(3, int), logits=True)
    assert np.array_equal(a, b)                       # the same context, in other pages
    m.close()


def test_lengths_follow_the_enqueued_steps(llm, orc):
    m, toks = start(llm, orc)
    m.batch_set([toks[70], toks[0]], [70, 0], [0, 1])
    assert [m.cache_length(s) for s in range(2)] == [70, 0]
    m.batch_enqueue()
    assert [m.cache_length(s) for s in range(2)] == [71, 1]
    m.batch_enqueue_decode(5)
    assert [m.cache_length(s) for s in range(2)] == [75, 5]
    m.batch_enqueue()
    m.batch_enqueue_decode(60)
    m.synchronize()
    assert [m.cache_length(s) for s in range(2)] == [135, 65] and m.cache_free_pages == 6 - 3 - 2
    with pytest.raises(RuntimeError):                 # past the pool: 72 more positions each want two pages
        m.batch_enqueue_decode(130)
    assert [m.cache_length(s) for s in range(2)] == [135, 65]
    m.close()


def test_enqueued_steps_do_not_wait_for_the_stream(llm, orc):
    """Steps enqueued behind work that takes long: the host goes on at once,
    across page ends and with pages shared until then, and what comes out is what
    the waiting calls give."""
    import time

    import torch
    m, toks = start(llm, orc, pages=16)
    start_at = np.array([toks[70], toks[71], 9], np.int32)
    m.cache_fork(0, 1, 70)
    m.cache_fork(0, 2, 64)
    want = m.generate_batch(start_at, [70, 70, 64], 130)
    kept = [m.cache_read(l, s, 190) for l in range(2) for s in range(3)]
    for s in (1, 2):
        m.cache_fork(0, s, 70 if s == 1 else 64)
    m.cache_truncate(0, 70)
    m.batch_set(start_at, [70, 70, 64], [0, 1, 2])
    side = torch.cuda.ExternalStream(m.stream)
    took = []
    for steps in (30, 30, 70):
        with torch.cuda.stream(side):
            torch.cuda._sleep(800_000_000)            # some 0.4 s
        t = time.perf_counter()
        m.batch_enqueue_decode(steps)
        took.append(time.perf_counter() - t)
    m.batch_enqueue()
    m.synchronize()
    assert max(took) < 0.2, took
    assert [m.cache_length(s) for s in range(3)] == [201, 201, 195]
    again = [m.cache_read(l, s, 190) for l in range(2) for s in range(3)]
    assert all(np.array_equal(a[i], b[i]) for a, b in zip(kept, again) for i in (0, 1))
    assert want.shape == (130, 3)
    m.close()


@pytest.mark.parametrize("paged", [True, False])
def test_what_a_refused_generation_reports(llm, orc, paged):
    """Past the context: a bad argument with either cache; past the pool: no memory."""
    from catseye_b200 import _lib
    m, toks = start(llm, orc)
    lib, ids = _lib.load(), np.zeros(1000, np.int32)
    if not paged:
        m.cache_q4(0)
    t, p = np.array([5], np.int32), np.array([70 if paged else 0], np.int32)
    run = lambda steps: lib.cats_gpu_llm_generate_batch(m.h, t.ctypes.data, p.ctypes.data, 1, steps, ids.ctypes.data)  # noqa: E731
    assert run(321) == 2
    if paged:
        m.cache_fork(0, 1, 70)
        m.cache_fork(0, 2, 70)
        m.batch_set([5, 6, 7], [70, 70, 70], [0, 1, 2])
        assert lib.cats_gpu_llm_batch_enqueue_decode(m.h, 251) == 2
        assert lib.cats_gpu_llm_batch_enqueue_decode(m.h, 180) == 3
    lib.cats_gpu_clear_error()
    assert run(3) == 0
    m.close()


@pytest.mark.parametrize("paged", [True, False])
def test_a_set_batch_goes_with_the_buffers_it_was_set_in(llm, orc, paged):
    """Larger buffers hold no batch yet; those that stay keep theirs."""
    m, toks = start(llm, orc)
    if not paged:
        m.cache_q4(0)
    m.batch_set(toks[:2], [0, 1], [0, 0])
    m.batch_reserve(64, 1)                            # not larger than what there is
    m.batch_enqueue()
    m.synchronize()
    m.batch_set(toks[:1], [0], [0])
    m.batch_reserve(300, 1)
    for call in (m.batch_enqueue, lambda: m.batch_enqueue_decode(1)):
        with pytest.raises(RuntimeError):
            call()
    m.batch_set(toks[:1], [0], [0])
    m.batch_enqueue_decode(2)
    m.synchronize()
    m.close()
