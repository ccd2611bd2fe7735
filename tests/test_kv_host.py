"""Paged Q4_0 KV cache, the parts that need no GPU: the page bookkeeping
(cats_gpu_kv_pages_*) against a model that copies token by token, and the
refusals of the device entry points, which come before any device call."""
import ctypes as C
import random

import numpy as np
import pytest

from catseye_b200 import _lib, kv

PAGE = kv.PAGE


class Model:
    """Sequences as lists of tokens; a pool of pages as lists."""

    def __init__(self, n_pages, n_seqs):
        self.seqs = [[] for _ in range(n_seqs)]
        self.pool = [[None] * PAGE for _ in range(n_pages)]

    def copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        got = [list(self.pool[s]) for s in src]
        for d, g in zip(dst, got):
            self.pool[d] = g

    def check(self, pages):
        table = pages.table()
        used = set()
        for s, want in enumerate(self.seqs):
            assert pages.length(s) == len(want)
            n = -(-len(want) // PAGE)
            assert (table[s, :n] >= 0).all() and (table[s, n:] == -1).all()
            used |= set(table[s, :n].tolist())
            assert [self.pool[table[s, i // PAGE]][i % PAGE] for i in range(len(want))] == want
        assert pages.free == len(self.pool) - len(used)


@pytest.mark.parametrize("seed", range(6))
def test_pages_hold_what_was_written(seed):
    r = random.Random(seed)
    n_pages, n_seqs, max_pages = r.choice([5, 24, 60]), 5, 9
    pages, m = kv.Pages(n_pages, n_seqs, max_pages), Model(n_pages, n_seqs)
    refused = written = 0
    for step in range(400):
        s = r.randrange(n_seqs)
        have = m.seqs[s]
        op = r.random()
        if op < 0.5:
            pos = r.choice([len(have), r.randint(0, len(have))])
            n = r.choice([0, 1, 2, 63, 64, 65, 150])
            before = pages.table()
            try:
                src, dst = pages.write(s, pos, n)
            except _lib.CatsGpuError as e:
                assert "memory" in str(e) or pos + n > max_pages * PAGE
                assert np.array_equal(before, pages.table())
                refused += 1
                continue
            m.copy(src.tolist(), dst.tolist())
            new = [(step, i) for i in range(n)]
            m.seqs[s] = have[:pos] + new + have[pos + n:]
            row = pages.table()[s]
            for i, v in zip(range(pos, pos + n), new):
                m.pool[row[i // PAGE]][i % PAGE] = v
            written += n
        elif op < 0.7:
            d = r.randrange(n_seqs)
            n = r.randint(0, len(have))
            if d == s:
                with pytest.raises(_lib.CatsGpuError):
                    pages.fork(s, d, n)
                continue
            pages.fork(s, d, n)
            m.seqs[d] = have[:n]
        elif op < 0.9:
            n = r.choice([0, r.randint(0, len(have))])
            pages.truncate(s, n)
            m.seqs[s] = have[:n]
        else:
            src, dst = pages.compact()
            m.copy(src.tolist(), dst.tolist())
            used = n_pages - pages.free
            assert pages.table().max(initial=-1) < used
        m.check(pages)
    assert written > 500 and (n_pages > 50 or refused)


def test_fork_copies_only_when_written():
    p = kv.Pages(8, 3, 4)
    p.write(0, 0, 100)
    p.fork(0, 1, 100)
    assert p.free == 6                               # both pages shared
    src, dst = p.write(1, 100, 1)                    # the partial one is copied, the whole one is not
    assert (src.tolist(), dst.tolist(), p.free) == ([1], [2], 5)
    src, _ = p.write(0, 100, 1)                      # nobody shares it any more
    assert src.size == 0
    p.truncate(0, 64)
    assert p.free == 6
    src, dst = p.write(0, 10, 1)                     # overwriting inside the shared whole page
    assert (src.tolist(), dst.tolist()) == ([0], [1])


def test_pages_refusals():
    lib = _lib.load()
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (-3, 2, 2), (1, 1, 1 << 30)):
        assert not lib.cats_gpu_kv_pages_create(*args)
        lib.cats_gpu_clear_error()
    p = kv.Pages(4, 2, 2)
    for seq, pos, n in ((2, 0, 1), (-1, 0, 1), (0, 1, 1), (0, -1, 1), (0, 0, -1), (0, 0, 129), (0, 0, 2**31 - 1)):
        with pytest.raises(_lib.CatsGpuError):
            p.write(seq, pos, n)
    p.write(0, 0, 128)
    p.write(1, 0, 128)
    assert p.free == 0
    for bad in (lambda: p.fork(0, 1, 129), lambda: p.fork(0, 2, 1), lambda: p.truncate(0, 129),
                lambda: p.truncate(0, -1), lambda: p.truncate(5, 0)):
        with pytest.raises(_lib.CatsGpuError):
            bad()
    assert p.length(0) == p.length(1) == 128 and p.length(7) == -1


def test_page_bytes():
    assert kv.page_bytes(1, 1, 128) == 64 * 2 * 128 * 9 // 16
    assert kv.page_bytes(80, 8, 128) == 80 * 8 * 9216
    for bad in ((1, 1, 48), (1, 1, 160), (0, 1, 64), (1, 0, 64), (1, 1, 0)):
        with pytest.raises(ValueError):
            kv.page_bytes(*bad)


# ---- refusals of the device entry points: nothing is launched, so the
# pointers need not be the device's
A = 1 << 20   # a 16-byte aligned address that is never followed
GOOD = dict(pool=A, table=A, n_pages=4, n_layers=2, n_kv_heads=2, head_size=64, n_seqs=2, max_pages=3)


def _call(name, cache, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(C.addressof(cache) if cache is not None else None, *args)
    lib.cats_gpu_clear_error()
    return rc


ROWS = dict(layer=0, k=A, v=A, type=0, ld_k=128, ld_v=128, rows=3, runs=A, n_runs=1, max_rows=3, stream=None)
ATT = dict(layer=0, out=A, q=2 * A, type=0, n_heads=4, ld_out=256, ld_q=256, rows=3, runs=A, n_runs=1, max_rows=3,
           max_len=5, stream=None)
BAD_CACHE = [dict(pool=0), dict(pool=A + 8), dict(table=0), dict(n_pages=0), dict(n_layers=0), dict(n_kv_heads=0),
             dict(head_size=48), dict(head_size=0), dict(head_size=-32), dict(n_seqs=0), dict(max_pages=0),
             dict(max_pages=1 << 26)]


@pytest.mark.parametrize("change", BAD_CACHE)
def test_bad_caches_are_refused(change):
    c = _lib.KvC(**{**GOOD, **change})
    for name, args in (("cats_gpu_kv_append_dev", ROWS), ("cats_gpu_kv_read_dev", ROWS),
                       ("cats_gpu_kv_attention_dev", ATT)):
        assert _call(name, c, *args.values()) == 2, name


@pytest.mark.parametrize("change", [dict(layer=-1), dict(layer=2), dict(k=0), dict(v=0), dict(k=A + 2), dict(type=2),
                                    dict(type=5), dict(ld_k=127), dict(ld_v=0), dict(rows=-1), dict(runs=0),
                                    dict(n_runs=-1), dict(max_rows=-1)])
def test_bad_rows_are_refused(change):
    args = {**ROWS, **change}
    for name in ("cats_gpu_kv_append_dev", "cats_gpu_kv_read_dev"):
        assert _call(name, _lib.KvC(**GOOD), *args.values()) == 2, name


@pytest.mark.parametrize("change", [dict(layer=2), dict(out=0), dict(q=0), dict(q=A + 1), dict(type=8), dict(n_heads=0),
                                    dict(n_heads=3), dict(n_heads=-2), dict(ld_out=255), dict(ld_q=1), dict(rows=-5),
                                    dict(runs=0), dict(n_runs=-1), dict(max_rows=-1), dict(max_len=-1)])
def test_bad_attention_is_refused(change):
    assert _call("cats_gpu_kv_attention_dev", _lib.KvC(**GOOD), *{**ATT, **change}.values()) == 2


def test_attention_over_its_own_queries_is_refused():
    assert _call("cats_gpu_kv_attention_dev", _lib.KvC(**GOOD), *{**ATT, "q": ATT["out"]}.values()) == 2


def test_rows_read_into_one_tensor_are_refused():
    assert _call("cats_gpu_kv_read_dev", _lib.KvC(**GOOD), *ROWS.values()) == 2


def test_large_heads_are_unsupported_and_nothing_is_nothing():
    big = _lib.KvC(**{**GOOD, "head_size": 256})
    assert _call("cats_gpu_kv_append_dev", big, *ROWS.values()) == 5
    assert _call("cats_gpu_kv_attention_dev", big, *ATT.values()) == 5
    c = _lib.KvC(**GOOD)
    assert _call("cats_gpu_kv_append_dev", None, *ROWS.values()) == 2
    for zero in (dict(rows=0), dict(n_runs=0)):
        assert _call("cats_gpu_kv_append_dev", c, *{**ROWS, **zero}.values()) == 0
        assert _call("cats_gpu_kv_attention_dev", c, *{**ATT, **zero}.values()) == 0


@pytest.mark.parametrize("src,dst", [([0], [4]), ([0], [-1]), ([4], [0]), ([-1], [0]), ([0, 1], [2, 2]), ([0], [0]),
                                     ([0, 1], [1, 2]), ([0, 0, 0, 0, 0], [1, 2, 3, 1, 2])])
def test_bad_page_copies_are_refused(src, dst):
    s, d = np.array(src, np.int32), np.array(dst, np.int32)
    c = _lib.KvC(**{**GOOD, "table": 0})
    assert _call("cats_gpu_kv_copy_pages_dev", c, s.ctypes.data, d.ctypes.data, len(src), None) == 2
    assert _call("cats_gpu_kv_copy_pages_dev", c, s.ctypes.data, d.ctypes.data, 0, None) == 0
    assert _call("cats_gpu_kv_copy_pages_dev", c, None, d.ctypes.data, 1, None) == 2


LP = dict(logits=A, type=0, rows=2, vocab=10, ld=10, targets=A, k=3, logprob=A, entropy=A, top_ids=A, top_logprob=A,
          stream=None)


@pytest.mark.parametrize("change,rc", [(dict(logits=0), 2), (dict(logits=A + 2), 2), (dict(type=2), 2),
                                       (dict(rows=-1), 2), (dict(vocab=0), 2), (dict(ld=9), 2), (dict(k=-1), 2),
                                       (dict(k=33), 5), (dict(targets=0), 2), (dict(top_ids=0), 2),
                                       (dict(top_logprob=0), 2), (dict(rows=0), 0)])
def test_bad_logprobs_are_refused(change, rc):
    lib = _lib.load()
    assert lib.cats_gpu_logprobs_dev(*{**LP, **change}.values()) == rc
    lib.cats_gpu_clear_error()
