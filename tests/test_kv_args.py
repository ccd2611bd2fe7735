"""Arguments of catseye_b200.kv and .score that are refused before any device call."""
import ctypes as C

import numpy as np
import pytest

from catseye_b200 import kv


@pytest.mark.parametrize("bad,error", [(np.array([1.0, 2.0]), TypeError), (np.array([0.5]), TypeError), ([1.5], TypeError),
                                       (np.array([True]), TypeError), (np.array([2**32 + 5]), OverflowError),
                                       (np.array([-2**31 - 1]), OverflowError), ([2**32 + 5], OverflowError),
                                       (np.array([2**63], np.uint64), OverflowError), (np.zeros((1, 2), np.int32), ValueError)])
def test_page_lists_that_are_not_page_numbers(bad, error):
    with pytest.raises(error):
        kv._ints(bad)


@pytest.mark.parametrize("good", [[3, -1, 7], (3, -1, 7), np.array([3, -1, 7]), np.array([3, -1, 7], np.int8),
                                  np.array([3, 0, -1, 0, 7, 0], np.int32)[::2]])
def test_page_lists(good):
    at, n, owner = kv._ints(good)
    assert n == 3 and list((C.c_int * 3).from_address(at)) == [3, -1, 7] and owner is not None
    assert kv._ints([])[1] == kv._ints(np.array([]))[1] == 0


def test_tensors_that_want_a_gradient():
    """Nothing silently stops a gradient; without one being recorded the same tensors pass."""
    import torch
    from catseye_b200 import score
    x, cpu = torch.zeros(2, 1, 32, requires_grad=True), torch.device("cpu")
    for call in (lambda: kv._rows(x, 1, 32, cpu, "k"), lambda: kv._rows(x * 2, 1, 32, cpu, "q"),
                 lambda: score.logprobs(torch.zeros(2, 5, requires_grad=True))):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        assert kv._rows(x, 1, 32, cpu, "k") == 32
    assert kv._rows(x.detach(), 1, 32, cpu, "k") == 32


@pytest.mark.parametrize("tp", [1, 2])
def test_rows_of_a_rank_hold_its_own_heads(tp):
    """cache_read of a tensor-parallel rank: the arrays it hands over are its kv heads' wide."""
    from catseye_b200 import llm

    class Lib:
        def cats_gpu_llm_cache_read(self, h, layer, seq, n, k, v):
            for i, p in enumerate((k, v)):
                C.memset(p.value, i + 1, n * 128 // tp * 4)
            return 0

    m = llm.GpuLLM.__new__(llm.GpuLLM)
    m.lib, m.h, m._tp_size = Lib(), None, tp
    m.cfg = llm.LlmConfig(dim=256, hidden=256, n_layers=1, n_heads=8, n_kv_heads=4, vocab=512, seq_len=64, wtype=2)
    k, v = m.cache_read(0, 0, 5)
    assert k.shape == v.shape == (5, 128 // tp)
    assert (k.view(np.uint8) == 1).all() and (v.view(np.uint8) == 2).all()


def test_page_bookkeeping_refuses_what_c_would_wrap():
    p = kv.Pages(4, 2, 3)
    p.write(0, 0, 70)
    big = 2**32
    for call in (lambda: p.write(0, big, 1), lambda: p.write(big, 70, 1), lambda: p.write(0, 70, big + 1),
                 lambda: p.fork(0, big + 1, 10), lambda: p.fork(big, 1, 10), lambda: p.fork(0, 1, big + 10),
                 lambda: p.truncate(0, big), lambda: p.truncate(big, 0), lambda: p.length(big),
                 lambda: kv.Pages(big + 1, 1, 1)):
        with pytest.raises(OverflowError):
            call()
    assert p.length(0) == 70 and p.length(1) == 0 and p.free == 2
