"""Attention over the paged Q4_0 cache where a call leaves the ordinary: rows
behind the table, values that are NaN, sums over very long sequences, very many
runs."""
import math

import numpy as np
import pytest
import torch

from catseye_b200 import _lib
from test_gpu_kv import LONG, TYPES, check_attention, fill, make, randn, runs_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(gpu):
    gpu.cats_gpu_clear_device_error()
    yield
    torch.cuda.synchronize()
    gpu.cats_gpu_clear_device_error()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mul,hint", [(1, 128), (3, 128), (1, LONG), (3, LONG)])
def test_rows_past_the_table_beside_a_nan(dtype, mul, hint):
    """A run that goes on past its sequence's table, its last position inside
    holding NaN: the rows behind it are zeros, not what lies behind the table."""
    c = make([128, 64], 1, 64)
    fill(c, [128, 64])
    v = randn(1, 1, 64, seed=4)
    v[0, 0, 5] = math.nan
    c.append(1, randn(1, 1, 64, seed=5), v, runs_of([(0, 1, 0, 127)]), 1)
    q = randn(4, mul, 64, seed=6).to(dtype)
    out = torch.full_like(q, 3)
    c.attention(1, out, q, runs_of([(0, 4, 0, 126)]), 4, hint)
    torch.cuda.synchronize()
    check_attention(c, 1, q, out, [(0, 1, 0, 126)], mul)
    o = out.double().cpu().numpy()
    assert np.isnan(o[1, :, :32]).all() and np.isfinite(o[1, :, 32:]).all()
    assert (o[2:] == 0).all()
    assert _lib.load().cats_gpu_device_error() == 0x40


def with_nan(lens, n_kv, hs, at):
    """Two caches that differ in the value rows named by `at` (sequence, position, head, element) only: NaN there."""
    clean, dirty = (make(lens, n_kv, hs, layers=1) for _ in range(2))
    for c in (clean, dirty):
        fill(c, lens)
    k, v = kv_rows(lens, n_kv, hs)
    for s, p, h, e in at:
        v[sum(lens[:s]) + p, h, e] = math.nan
    first = np.cumsum([0] + list(lens[:-1]))
    dirty.append(0, k, v, runs_of([(int(f), n, i, 0) for i, (f, n) in enumerate(zip(first, lens))]), max(lens))
    return clean, dirty


def kv_rows(lens, n_kv, hs):
    return randn(sum(lens), n_kv, hs, seed=0), randn(sum(lens), n_kv, hs, seed=1)   # as fill() makes them


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,mul", [(32, 1), (64, 4), (96, 2), (128, 8), (128, 1)])
@pytest.mark.parametrize("new,lens,hint", [([300], [700], None), ([700, 1, 9], [700, 150, 400], None), ([1, 3], [400, 300], None),
                                           ([20, 1, 3], [700, 150, 400], (20, LONG))])
def test_a_nan_is_only_where_it_is_seen(dtype, hs, mul, new, lens, hint):
    """NaN in some value rows, first and last of a page, of a tile and of a run:
    rows that see one are NaN in its block of 32, and all else is, bit for
    bit, what the cache without them gives."""
    n_kv = 2
    at = [(s, p, h, e) for s, n in enumerate(lens)
          for p, h, e in ((n - 1, 0, 3), (n - new[s], 1, hs - 1), (n - max(new[s] // 2, 1), 0, hs // 2), (128, 1, 0)) if 0 <= p < n]
    clean, dirty = with_nan(lens, n_kv, hs, at)
    rows, first, runs = sum(new), 0, []
    for i, (n, m) in enumerate(zip(new, lens)):
        runs.append((first, n, i, m - n))
        first += n
    q = randn(rows, n_kv * mul, hs, seed=9).to(dtype)
    want, got = torch.full_like(q, 3), torch.full_like(q, 3)
    for c, o in ((clean, want), (dirty, got)):
        c.attention(0, o, q, runs_of(runs), *(hint or (max(new), max(lens))))
    bad = torch.zeros(rows, n_kv * mul, hs // 32, dtype=torch.bool)
    for f, n, s, pos in runs:
        for t, p, h, e in at:
            if t == s:
                bad[f + max(p - pos, 0):f + n, h * mul:(h + 1) * mul, e // 32] = True
    bad = bad.repeat_interleave(32, 2)
    got, want = got.cpu(), want.cpu()
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [8000, 5])
def test_a_nan_does_not_stall_the_batch(dtype, new):
    """A value row of NaN in every page of a long sequence: the call takes about as long as without."""
    lens = [8000]
    clean, dirty = with_nan(lens, 2, 128, [(0, p, h, e) for p in range(7, 8000, 64) for h in (0, 1) for e in (0, 40, 80, 127)])
    q = randn(new, 8, 128, seed=2).to(dtype)
    out = torch.empty_like(q)
    took = []
    for c in (clean, dirty):
        each = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            c.attention(0, out, q, runs_of([(0, new, 0, 8000 - new)]), new, 8000)
            b.record()
            torch.cuda.synchronize()
            each.append(a.elapsed_time(b))
        took.append(sorted(each)[2])
    assert took[1] < 2 * took[0] + 0.05, took


@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("rows,hint", [(1, (1, 1)), (8, (8, 1)), (1, (1, LONG)), (60, (60, 140000)), (300, (300, 140000))])
def test_long_sums_of_fp32_rows_are_rounded(hs, rows, hint):
    """131072 values of one sign under nearly flat probabilities, independent of
    them: what is off is the sums.  A warp adds 32768 tokens, 16 at a time: 2048
    additions to a sum that grows evenly.  Rounded, each is off by 2^-24 of the
    sum so far at most, 2^-24 / sqrt(3) rms; over the additions that is
    sqrt(2048 / 3) 2^-24 / sqrt(3) = 9e-7 of the mean, and the sum of the
    probabilities as much again: sqrt(2) 9e-7.  What is off in single
    probabilities (2^-21 each) averages out.  Six such deviations cover some
    thousand outputs; parts that are joined are off by less.  (Cut off instead of
    rounded the additions are all off the same way: some 2048 2^-26 = 3e-5.)"""
    n = 131072
    c = make([n], 1, hs, layers=1)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = torch.randn(n, 1, hs, generator=g, device="cuda"), torch.rand(n, 1, hs, generator=g, device="cuda") + 0.5
    runs = runs_of([(0, n, 0, 0)])
    c.append(0, k, v, runs, n)
    c.read(0, k, v, runs, n)
    q = torch.randn(rows, 4, hs, generator=g, device="cuda") * 0.3
    out = torch.full_like(q, 3)
    c.attention(0, out, q, runs_of([(0, rows, 0, n - rows)]), *hint)
    k, v = k[:, 0].double(), v[:, 0].double()
    hidden = torch.arange(n, device="cuda") > torch.arange(n - rows, n, device="cuda")[:, None]
    for h in range(4):
        p = torch.softmax((q[:, h].double() @ k.T / math.sqrt(hs)).masked_fill(hidden, -math.inf), 1)
        off = (out[:, h].double() / (p @ v) - 1).abs().max()
        assert off <= 6 * 2**0.5 * 9e-7, off


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,n_runs,long", [(32, 9000, 4300), (96, 700, 90), (64, 70000, 40)])
def test_many_runs_beside_a_long_one(dtype, hs, n_runs, long):
    """Thousands of runs of one row or none and a longer one, and a hint far past what the tensor holds."""
    n_kv, lens = 16, [long + 10, 30]
    c = make(lens, n_kv, hs, layers=1)
    fill(c, lens)
    single = [(long + i, 1, 1, 20 + i) for i in range(5)]
    runs = [(0, 0, 1, 0)] * 100 + single[:2] + [(0, long, 0, 10)] + [(0, 0, 0, 7)] * (n_runs - 106) + single[2:]
    q = randn(long + 6, n_kv, hs, seed=7).to(dtype)
    outs = []
    for hint in ((long, long + 10), (2**31 - 1, 2**31 - 1)):
        out = torch.full_like(q, 3)
        c.attention(0, out, q, runs_of(runs), *hint)
        outs.append(out)
    torch.cuda.synchronize()
    few = [(long, 1, 1, 20), (long + 4, 1, 1, 24), (0, 2, 0, 10), (long - 1, 1, 0, long + 9)]
    for out in outs:
        check_attention(c, 0, q, out, few, 1)
        assert (out[long + 5:] == 3).all() and out[:long + 5].isfinite().all()
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("hs", [32, 64, 96, 128])
@pytest.mark.parametrize("rows,mul,hint", [(1, 4, (1, 1)), (8, 4, (8, 1)), (1, 4, (1, LONG)), (60, 4, (60, 140000))])
def test_long_sums_of_fp16_rows_are_not_cut_off(hs, rows, mul, hint):
    long_fp16_sums(hs, rows, mul, hint, 131072)


def long_fp16_sums(hs, rows, mul, hint, n):
    """The same for fp16 rows, where the outputs' roundings hide single sums but
    not their mean: an output is off by 2^-11 / sqrt(12) of itself rms at most
    (its rounding), 1.4e-4, so the mean of 4 hs outputs by 1.4e-4 / sqrt(4 hs);
    six of those.  What the sums are cut off by goes one way: accumulators hold
    the products of 4096 tokens at most before they are added, rounded, to the
    rest; 256 products of 2^-23 lose 2^-16 on average over them as they grow."""
    c = make([n], 1, hs, layers=1)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = torch.randn(n, 1, hs, generator=g, device="cuda"), torch.rand(n, 1, hs, generator=g, device="cuda") + 0.5
    runs = runs_of([(0, n, 0, 0)])
    c.append(0, k, v, runs, n)
    c.read(0, k, v, runs, n)
    q = (torch.randn(rows, mul, hs, generator=g, device="cuda") * 0.3).half()
    out = torch.full_like(q, 3)
    c.attention(0, out, q, runs_of([(0, rows, 0, n - rows)]), *hint)
    k, v = k[:, 0].double(), v[:, 0].double()
    hidden = torch.arange(n, device="cuda") > torch.arange(n - rows, n, device="cuda")[:, None]
    off = []
    for h in range(4):
        p = torch.softmax((q[:, h].double() @ k.T / math.sqrt(hs)).masked_fill(hidden, -math.inf), 1)
        off.append(out[:, h].double() / (p @ v) - 1)
    off = torch.stack(off).mean()
    assert off.abs() <= 6 * 1.4e-4 / math.sqrt(4 * hs) + 2**-16, off


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("n", [16384, 131072, 4096, 4097, 8192 + 77])
def test_long_sums_of_fp16_prompts_are_not_cut_off(hs, n):
    """The same for prompts, at lengths around the ends of what one accumulator takes."""
    long_fp16_sums(hs, 300, 16, (300, n), n)
