"""Paged Q4_0 KV cache on the GPU (catseye_b200.kv) against its definition in
64 bits: blocks written and read back, causal attention over ragged batches,
page copies, and the runs they form together.

Tolerances.  The values a cache holds are exact in fp32 and fp16, so append
and read are compared for equality.  Attention of a row: with B = max over
positions of sum_i |q_i k_i| / sqrt(hs), a score is off by at most
B (hs + 8) 2^-24 (sums in fp32) + B 2^-21 (q as two fp16 halves of 11 bits each,
the exponential's argument), which enters a probability's exponent, so the
softmax weights are off by 2x that relative; the probabilities as two fp16
halves add 2^-21, the exponentials 2^-20, and the weighted sum's additions
n 2^-24, all times max |v|.  fp16 and bf16 rows: the probabilities are rounded
once to fp16 (2^-11 max |v|, twice as the normaliser is not rounded alike),
bf16 query rows lie exactly in fp16's range after scaling, and the output is
rounded by half a step."""
import math
import os
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

from catseye_b200 import _lib, kv

pytestmark = pytest.mark.gpu
PAGE = 64
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _clean(gpu):
    gpu.cats_gpu_clear_device_error()
    yield
    torch.cuda.synchronize()
    gpu.cats_gpu_clear_device_error()


def blocks(x):
    """The values Q4_0 blocks stand for, float64 (the definition, in 64 bits)."""
    x = np.asarray(x, np.float64)
    shape = x.shape
    x = x.reshape(-1, 32)
    hi, lo = x.max(1), x.min(1)
    m = np.where(hi >= -lo, hi, lo)
    frac, e = np.frexp(-m / 8)
    d = np.ldexp(np.round(frac * 256) / 256, e)
    d = np.clip(d, -8160, 8160).astype(np.float16).astype(np.float64)[:, None]
    with np.errstate(all="ignore"):
        code = np.clip(np.floor(np.where(d == 0, 0, x / np.where(d == 0, 1, d)) + 0.5), -8, 7)
    out = code * d
    out[~np.isfinite(x).all(1)] = np.nan
    return out.reshape(shape)


def held(cache, layer, seq, n):
    """K and V rows 0..n-1 of a sequence as the documented layout holds them, float64."""
    hs, hb = cache.head_size, cache.head_size // 32
    table, pool = cache.table.cpu().numpy(), cache.pool.cpu().numpy()
    t = np.arange(n)
    chunk = pool[table[seq, t // PAGE], layer]                  # [n, heads, bytes]
    half = np.ascontiguousarray(chunk).view(np.float16).astype(np.float64)
    e, s = np.arange(hs)[None], (t % PAGE)[:, None]
    b, r = e // 32, e % 32
    at = lambda a, i: np.take_along_axis(a, np.broadcast_to(i[:, None], (n, a.shape[1], hs)), 2)  # noqa: E731
    k = at(chunk, s * 16 * hb + r // 8 * 4 * hb + 4 * b + r % 8 // 2) >> (r % 2 * 4)[None] & 15
    v = at(chunk, 1024 * hb + ((s // 2 * 8 + r // 4) * hb + b) * 4 + s % 2 * 2 + r % 4 // 2) >> (r % 2 * 4)[None] & 15
    return ((k.astype(np.float64) - 8) * at(half, 1024 * hb + s * hb + b),
            (v.astype(np.float64) - 8) * at(half, 1088 * hb + (s // 2 * hb + b) * 2 + s % 2))


def make(lens, n_kv, hs, layers=2, seed=0, spare=3):
    """A cache with NaN-like bytes everywhere and room for `lens` tokens of each sequence, pages in random order."""
    need = [-(-n // PAGE) for n in lens]
    c = kv.Cache.empty(sum(need) + spare, layers, n_kv, hs, len(lens), max(max(need), 1))
    c.pool.fill_(255)
    order = np.random.default_rng(seed).permutation(sum(need) + spare)
    t = np.full(tuple(c.table.shape), -1, np.int32)
    for i, n in enumerate(need):
        t[i, :n], order = order[:n], order[n:]
    c.table.copy_(torch.from_numpy(t))
    return c


def runs_of(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda").reshape(-1, 4)


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------ append and read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,n_kv", [(32, 1), (64, 3), (96, 2), (128, 8)])
def test_append_and_read_hold_the_definition(dtype, hs, n_kv):
    """Ragged runs, some behind earlier rows, one empty: the cache's bytes and read() give the blocks' values."""
    new, past = [1, 70, 0, 64, 5], [0, 37, 12, 64, 127]
    c = make([n + p for n, p in zip(new, past)], n_kv, hs, layers=3)
    rows = sum(new)
    k = randn(rows, n_kv, hs, seed=1, dtype=dtype) * 3
    v = randn(rows, n_kv, hs, seed=2, dtype=dtype) * torch.exp(randn(n_kv, hs, seed=3)).to(dtype)
    first, runs = 0, []
    for i, (n, p) in enumerate(zip(new, past)):
        runs.append((first, n, i, p))
        first += n
    before = c.pool.clone()
    c.append(1, k, v, runs_of(runs), max(new))
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    c.read(1, kb, vb, runs_of(runs), max(new))
    for got, x in ((kb, k), (vb, v)):
        want = torch.from_numpy(blocks(x.double().cpu().numpy())).to(dtype)
        assert torch.equal(got.cpu(), want)
    for f, n, s, p in runs:
        if n:
            hk, hv = held(c, 1, s, n + p)
            assert np.array_equal(hk[p:], blocks(k[f:f + n].double().cpu().numpy()))
            assert np.array_equal(hv[p:], blocks(v[f:f + n].double().cpu().numpy()))
    assert torch.equal(c.pool[:, 0], before[:, 0]) and torch.equal(c.pool[:, 2], before[:, 2])
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_quantizer_at_its_borders(dtype):
    """Values next to and on the borders between codes, blocks of zeros, of one
    sign, of both extremes, tiny, subnormal, saturating, and non-finite ones."""
    d = np.float32(0.40625)
    rows = []
    for step in (-2, -1, 0, 1, 2):
        x = (np.arange(32, dtype=np.float32) % 15 - 7.5) * d
        x = np.array([np.nextafter(a, np.float32(np.sign(step) * np.inf)) if step else a for a in x], np.float32)
        if abs(step) == 2:
            x = np.nextafter(x, np.float32(np.sign(step) * np.inf))
        x[0] = -8 * d
        rows.append(x)
        y = x.copy()
        y[0] = 8 * d                                             # a negative scale
        rows.append(y)
        z = y.copy()
        z[1] = -8 * d                                            # both signs reach it
        rows.append(z)
    rng = np.random.default_rng(0)
    base = rng.standard_normal(32).astype(np.float32)
    rows += [np.zeros(32), -np.zeros(32), np.abs(base), -np.abs(base), base * 1e-7, base * 3e-8, base * 1e-38,
             base * 1e-42, base * 2e4, base * 1e5, base * 1e30, np.full(32, 65504.), np.full(32, -3e38)]
    for bad in (np.nan, np.inf, -np.inf):
        b = base.copy()
        b[rng.integers(32)] = bad
        rows.append(b)
    x = torch.tensor(np.array(rows, np.float32), device="cuda").to(dtype)[:, None]          # [n, 1, 32]
    n = x.shape[0]
    c = make([n], 1, 32, layers=1)
    run = runs_of([(0, n, 0, 0)])
    c.append(0, x, x, run, n)
    k, v = torch.empty_like(x), torch.empty_like(x)
    c.read(0, k, v, run, n)
    want = torch.from_numpy(blocks(x.double().cpu().numpy())).to(dtype).double().numpy()
    assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(v.double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1, -1])
def test_quantizer_on_every_16_bit_value(dtype, sign):
    """Every finite value in blocks of every significand a scale can have, at
    scales that make it small, large, out of range and subnormal."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every.float())]
    for top in [sign * 8 * s * (128 + i) / 128 for i in range(0, 128, 5 if sign < 0 else 3) for s in (1.0,)] + \
            [sign * 2.0 ** e for e in (-24, -16, -14, 9, 13, 15)]:
        x = every[(every.abs() <= abs(torch.tensor(top).to(dtype).float())) & (every.abs() >= abs(top) * 2.0**-6)]
        x = torch.nn.functional.pad(x, (0, -x.numel() % 31)).view(-1, 31)
        x = torch.cat([torch.full((len(x), 1), top, dtype=dtype), x], 1)[:, None].cuda()    # [n, 1, 32]
        n = x.shape[0]
        c = make([n], 1, 32, layers=1)
        run = runs_of([(0, n, 0, 0)])
        c.append(0, x, x.flip(2), run, n)
        k, v = torch.empty_like(x), torch.empty_like(x)
        c.read(0, k, v, run, n)
        assert torch.equal(k.cpu(), torch.from_numpy(blocks(x.double().cpu().numpy())).to(dtype)), top
        assert torch.equal(v.cpu(), torch.from_numpy(blocks(x.flip(2).double().cpu().numpy())).to(dtype)), top


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_rows_of_a_wider_tensor(dtype, shift):
    """k and v as slices of a qkv row (any alignment), read back into slices; what lies between stays."""
    n, n_kv, hs = 37, 2, 64
    x = randn(n, 7 * hs + shift + 3, seed=4, dtype=dtype)
    k = x[:, shift:shift + 2 * hs].unflatten(1, (n_kv, hs))
    v = x[:, shift + 3 * hs:shift + 5 * hs].unflatten(1, (n_kv, hs))
    c = make([n], n_kv, hs)
    run = runs_of([(0, n, 0, 0)])
    c.append(0, k, v, run, n)
    back = torch.full_like(x, 5)
    c.read(0, back[:, shift:shift + 2 * hs].unflatten(1, (n_kv, hs)),
           back[:, shift + 3 * hs:shift + 5 * hs].unflatten(1, (n_kv, hs)), run, n)
    want = torch.full_like(x, 5)
    want[:, shift:shift + 2 * hs] = torch.from_numpy(blocks(k.double().cpu().numpy())).to(dtype).flatten(1).cuda()
    want[:, shift + 3 * hs:shift + 5 * hs] = torch.from_numpy(blocks(v.double().cpu().numpy())).to(dtype).flatten(1).cuda()
    assert torch.equal(back, want)


def test_what_lies_outside_is_left_out():
    """Runs that name rows, sequences, positions or pages outside their range:
    nothing is written there, rows read from there are zeros, a bit is set."""
    n_kv, hs = 1, 32
    lib = _lib.load()
    c = make([100, 64], n_kv, hs, layers=1)
    x = randn(8, n_kv, hs, seed=5)
    before = c.pool.clone()
    for run in ((0, 4, 2, 0), (0, 4, -1, 0), (0, 4, 0, 128), (0, 4, 0, -4), (0, 4, 1, 64), (8, 4, 0, 0), (-4, 4, 0, 0)):
        c.append(0, x, x, runs_of([run]), 4)
        torch.cuda.synchronize()
        assert lib.cats_gpu_device_error() == 0x40, run
        assert torch.equal(c.pool, before), run
        k, v = torch.full_like(x, 7), torch.full_like(x, 7)
        c.read(0, k, v, runs_of([run]), 4)
        assert (k[:4] == 0).all() == (0 <= run[0] < 8) and (k[4:] == 7).all(), run
        lib.cats_gpu_clear_device_error()
    c.table[0, 0] = c.n_pages                        # a page past the pool
    before = c.pool.clone()
    c.append(0, x, x, runs_of([(0, 4, 0, 0)]), 4)
    assert torch.equal(c.pool, before) and lib.cats_gpu_device_error() == 0x40


def test_launch_hints_smaller_than_the_batch():
    """max_rows below the longest run costs time, not rows."""
    c = make([500], 2, 64)
    x = randn(500, 2, 64, seed=6)
    k, v = torch.empty_like(x), torch.empty_like(x)
    c.append(0, x, x, runs_of([(0, 500, 0, 0)]), 1)
    c.read(0, k, v, runs_of([(0, 500, 0, 0)]), 0)
    assert np.array_equal(k.double().cpu().numpy(), blocks(x.double().cpu().numpy()))


# ---------------------------------------------------------------- attention
def check_attention(c, layer, q, out, runs, mul, untouched=None):
    """Every row of every run against float64, within the bound of the module's text."""
    hs, dtype = c.head_size, q.dtype
    qd, od = q.double().cpu().numpy(), out.double().cpu().numpy()
    half = torch.finfo(dtype).eps / 2
    covered = np.zeros(q.shape[0], bool)
    worst = 0.0
    for first, n, seq, pos in runs:
        if n <= 0:
            continue
        k, v = held(c, layer, seq, max(pos + n, 1))
        for i in range(n):
            covered[first + i] = True
            seen = pos + i + 1
            if seen <= 0:
                assert (od[first + i] == 0).all()
                continue
            for h in range(q.shape[1]):
                kk, vv = k[:seen, h // mul], v[:seen, h // mul]
                s = kk @ qd[first + i, h] / math.sqrt(hs)
                p = np.exp(s - s.max())
                want = p @ vv / p.sum()
                big = (np.abs(kk) @ np.abs(qd[first + i, h])).max() / math.sqrt(hs)
                tol = 2 * big * ((hs + 8) * 2**-24 + 2**-21) + 2**-20 + 2**-21 + seen * 2**-24
                if dtype != torch.float32:
                    tol += 2 * 2**-11
                tol = tol * np.abs(vv).max() + half * np.abs(want)
                err = np.abs(od[first + i, h] - want)
                worst = max(worst, (err / tol).max())
                assert (err <= tol).all(), (first + i, h, (err / tol).max())
    if untouched is not None:
        assert (od[~covered] == untouched).all()
    return worst


def fill(c, lens, seed=0, scale=1.0):
    """Append random K/V for every sequence and layer."""
    rows = sum(lens)
    first, runs = 0, []
    for i, n in enumerate(lens):
        runs.append((first, n, i, 0))
        first += n
    for layer in range(c.n_layers):
        c.append(layer, randn(rows, c.n_kv_heads, c.head_size, seed=seed + 10 * layer) * scale,
                 randn(rows, c.n_kv_heads, c.head_size, seed=seed + 10 * layer + 1), runs_of(runs), max(lens))


def attend(c, layer, new, lens, mul, dtype, seed=9, extra=2, hints=None, sharp=1.0):
    rows = sum(new)
    first, runs = 0, []
    for i, (n, m) in enumerate(zip(new, lens)):
        runs.append((first, n, i, m - n))
        first += n
    q = (randn(rows + extra, c.n_kv_heads * mul, c.head_size, seed=seed) * sharp).to(dtype)
    out = torch.full_like(q, 3)
    mr, ml = hints or (max(new), max(lens))
    c.attention(layer, out, q, runs_of(runs), mr, ml)
    return q, out, runs


DECODE = [[1], [2, 63], [64, 65, 1], [127, 128, 129, 300, 5, 511, 512, 513], [1500]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,n_kv,mul", [(32, 1, 1), (64, 2, 3), (96, 1, 8), (128, 2, 1), (128, 1, 16), (128, 1, 20)])
@pytest.mark.parametrize("lens", DECODE)
def test_decode_attention(dtype, hs, n_kv, mul, lens):
    """One row a sequence; lengths around the pages' ends; rows behind the batch stay."""
    c = make(lens, n_kv, hs)
    fill(c, lens)
    q, out, runs = attend(c, 1, [1] * len(lens), lens, mul, dtype)
    check_attention(c, 1, q, out, runs, mul, untouched=3)
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,n_kv,mul", [(32, 2, 1), (64, 1, 3), (96, 1, 4), (128, 1, 1), (128, 1, 8)])
@pytest.mark.parametrize("new,lens", [([2], [2]), ([65], [65]), ([33, 0, 1, 7], [33, 40, 150, 71]), ([130], [260]),
                                      ([16, 17, 128], [80, 17, 129])])
def test_prompt_attention(dtype, hs, n_kv, mul, new, lens):
    """Runs of rows behind caches of other lengths, one empty."""
    c = make(lens, n_kv, hs)
    fill(c, lens)
    q, out, runs = attend(c, 0, new, lens, mul, dtype)
    check_attention(c, 0, q, out, runs, mul, untouched=3)


# A context of LONG tokens is planned as equal stretches over the whole GPU
# and a second kernel that joins them, whatever the runs' true lengths are.
LONG = 1_000_000


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs,n_kv,mul", [(32, 2, 1), (64, 1, 3), (96, 2, 4), (128, 2, 1), (128, 1, 8), (128, 1, 20)])
@pytest.mark.parametrize("lens", DECODE + [[5000, 1, 700]])
def test_decode_attention_in_stretches(dtype, hs, n_kv, mul, lens):
    c = make(lens, n_kv, hs)
    fill(c, lens)
    q, out, runs = attend(c, 1, [1] * len(lens), lens, mul, dtype, hints=(1, LONG))
    check_attention(c, 1, q, out, runs, mul, untouched=3)
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hint", [1, 3, 100])
@pytest.mark.parametrize("new,lens", [([2], [2]), ([33, 0, 1, 7], [33, 40, 150, 71]), ([1, 90, 20], [400, 90, 1000])])
def test_rows_in_stretches(dtype, hint, new, lens):
    """Runs of more and of fewer rows than the hint says, beside empty ones."""
    c = make(lens, 2, 64)
    fill(c, lens)
    q, out, runs = attend(c, 0, new, lens, 2, dtype, hints=(hint, LONG))
    check_attention(c, 0, q, out, runs, 2, untouched=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("new,lens", [([700], [1800]), ([300, 1, 0, 2, 1, 1, 5], [900, 1300, 10, 200, 64, 1, 517]),
                                      ([250, 250, 249], [250, 1250, 513])])
def test_long_prompts(dtype, hs, new, lens):
    """Rows for several tiles over several tiles of tokens; prompts beside single tokens."""
    c = make(lens, 4, hs)
    fill(c, lens)
    q, out, runs = attend(c, 1, new, lens, 4, dtype)
    check_attention(c, 1, q, out, runs, 4, untouched=3)
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_long_prompts_with_holes_and_nan(dtype):
    """A NaN value row seen by the last rows only, one that is not seen, a page
    that is missing, maxima that move late, rows before position 0."""
    lens = [900, 1400]
    c = make(lens, 4, 64)
    fill(c, lens)
    x = randn(64, 4, 64, seed=1)
    c.append(0, x * 8, x, runs_of([(0, 64, 0, 800)]), 64)             # large keys late in the sequence
    nan = torch.full_like(x, math.nan)
    c.append(0, x, nan, runs_of([(0, 1, 0, 100), (0, 1, 1, 1390)]), 1)
    q = randn(820, 16, 64, seed=3).to(dtype)
    out = torch.full_like(q, 3)
    runs = [(0, 400, 0, -320), (400, 400, 1, 1000), (800, 20, 0, 880)]
    c.attention(0, out, q, runs_of(runs), 400, 1400)
    o = out.double().cpu().numpy()
    assert (o[:320] == 0).all() and np.isfinite(o[:400]).all() and np.isfinite(o[400:790]).all()
    assert np.isnan(o[790:800]).all() and np.isnan(o[800:]).all()
    check_attention(c, 0, q, out, [(0, 400, 0, -320), (400, 390, 1, 1000)], 4)
    plain = torch.full_like(q, 3)
    c.table[1, 9] = -1
    c.attention(0, out, q, runs_of(runs[1:2]), 400, 1400)
    c.attention(0, plain, q, runs_of(runs[1:2]), 1, 1400)             # the other kernel, by its hint
    torch.cuda.synchronize()
    assert _lib.load().cats_gpu_device_error() == 0x40
    assert (out[400:790].float() - plain[400:790].float()).abs().max() < (2**-16 if dtype == torch.float32 else 2**-7)


@pytest.mark.parametrize("dtype", TYPES)
def test_stretches_with_holes_and_what_is_masked(dtype):
    """Missing pages, rows before position 0, a batch of empty runs, NaN behind the mask: in stretches as in one piece."""
    lens = [700, 300]
    c = make(lens, 1, 64)
    fill(c, lens)
    dead = randn(64, 1, 64, seed=1)
    dead[:] = math.nan
    c.append(0, dead, dead, runs_of([(0, 20, 0, 680), (0, 1, 1, 299)]), 20)   # rows 680.. and 299 are NaN
    q = randn(30, 2, 64, seed=3).to(dtype)
    for runs in ([(0, 10, 0, 670), (10, 1, 1, 298), (11, 0, 1, 0)], [(0, 12, 1, -5), (12, 4, 0, 0)],
                 [(0, 0, 0, 0), (3, 0, 1, 5)]):
        got = torch.full_like(q, 3)
        c.attention(0, got, q, runs_of(runs), 1, LONG)
        check_attention(c, 0, q, got, runs, 2, untouched=3)
    assert _lib.load().cats_gpu_device_error() == 0
    c.table[0, 3] = -1
    piece, stretch = torch.full_like(q, 3), torch.full_like(q, 3)
    c.attention(0, piece, q, runs_of([(0, 4, 0, 600)]), 4, 700)
    c.attention(0, stretch, q, runs_of([(0, 4, 0, 600)]), 4, LONG)
    assert torch.isfinite(stretch).all() and (piece.float() - stretch.float()).abs().max() < 2**-8
    torch.cuda.synchronize()
    assert _lib.load().cats_gpu_device_error() == 0x40


@pytest.mark.parametrize("rows,hint", [(1, LONG), (64, 2000), (1, 2000)])
def test_captured_replayed_and_on_two_streams(rows, hint):
    """One captured call replayed after its inputs moved on; two streams at once: each the answer of a call alone."""
    lens = [2000, 900]
    c = make(lens, 2, 128)
    fill(c, lens)
    runs = runs_of([(0, rows, 0, 2000 - rows), (rows, rows, 1, 900 - rows)])
    qs = [randn(2 * rows, 8, 128, seed=20 + i).half() for i in range(6)]
    alone = []
    for q in qs:
        alone.append(torch.empty_like(q))
        c.attention(0, alone[-1], q, runs, rows, hint)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [torch.empty_like(q) for q in qs]
    for i, q in enumerate(qs):
        c.attention(0, got[i], q, runs, rows, hint, stream=side[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, got))
    graphs, ins, outs = [], [], []
    for s in side:
        ins.append(qs[0].clone())
        outs.append(torch.empty_like(qs[0]))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            c.attention(0, outs[-1], ins[-1], runs, rows, hint, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for i in range(0, 6, 2):                          # both graphs in flight together
        for j in range(2):
            ins[j].copy_(qs[i + j])
        torch.cuda.synchronize()
        for j in range(2):
            with torch.cuda.stream(side[j]):
                graphs[j].replay()
                graphs[j].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j], alone[i + j])


FIRST = """
import torch
from catseye_b200 import kv
c = kv.Cache.empty(40, 1, 2, 64, 1, 40)
c.table.copy_(torch.arange(40, dtype=torch.int32)[None])
x = torch.randn(2000, 2, 64, device="cuda")
c.append(0, x, x, torch.tensor([[0, 2000, 0, 0]], dtype=torch.int32, device="cuda"), 2000)
q, out, want = (torch.randn(1, 8, 64, device="cuda") for _ in range(3))
run = torch.tensor([[0, 1, 0, 1999]], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=torch.cuda.Stream(), capture_error_mode="thread_local"):
    c.attention(0, out, q, run, 1, 1_000_000, stream=torch.cuda.current_stream().cuda_stream)
g.replay()
torch.cuda.synchronize()
c.attention(0, want, q, run, 1, 1_000_000)
torch.cuda.synchronize()
assert torch.equal(out, want)
"""


def test_the_first_call_of_a_process_is_captured():
    """Nothing the library makes once (attributes, memory pool) asks for an eager call first."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_rows_before_position_zero_see_nothing(dtype, rows):
    """A run that starts at a negative position: its first rows get zeros, the others see what there is."""
    c = make([rows + 3], 1, 64)
    fill(c, [rows + 3])
    q = randn(rows + 5, 2, 64, seed=3).to(dtype)
    out = torch.full_like(q, 3)
    runs = [(0, rows + 5, 0, -5)]
    c.attention(0, out, q, runs_of(runs), rows + 5, rows)
    check_attention(c, 0, q, out, runs, 2)
    assert _lib.load().cats_gpu_device_error() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 50])
def test_peaked_and_flat_rows(dtype, rows):
    """Scores in the hundreds (one position takes all) and all equal."""
    lens = [400]
    c = make(lens, 1, 128)
    fill(c, lens, scale=4.0)
    for sharp in (0.0, 8.0):
        q, out, runs = attend(c, 0, [rows], lens, 4, dtype, sharp=sharp)
        check_attention(c, 0, q, out, runs, 4, untouched=3)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e5, 1e8])
def test_magnitudes(rows, size):
    """Query rows far from 1 (beyond fp16 either way) against keys that bring the scores back."""
    lens, dtype = [150], torch.float32
    c = make(lens, 1, 64, layers=1)
    ks = min(max(1 / size, 1e-4), 1e3)
    c.append(0, randn(150, 1, 64, seed=1) * ks, randn(150, 1, 64, seed=2) * 1e-3, runs_of([(0, 150, 0, 0)]), 150)
    q = randn(rows, 3, 64, seed=3) * size
    out = torch.empty_like(q)
    runs = [(0, rows, 0, 150 - rows)]
    c.attention(0, out, q.to(dtype), runs_of(runs), rows, 150)
    check_attention(c, 0, q, out, runs, 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 30])
def test_nan_in_the_cache_reaches_the_rows_that_see_it(dtype, rows):
    """A NaN held at one position shows in every row that sees it and in no other; masked ones do not count."""
    lens = [100]
    c = make(lens, 2, 64, layers=1)
    k, v = randn(100, 2, 64, seed=1), randn(100, 2, 64, seed=2)
    v[80, 0, 3] = math.nan
    k[90, 1, 40] = math.inf
    c.append(0, k, v, runs_of([(0, 100, 0, 0)]), 100)
    q = randn(100, 4, 64, seed=3).to(dtype)
    out = torch.full_like(q, 3)
    runs = [(i, min(rows, 100 - i), 0, i) for i in range(0, 100, rows)]
    c.attention(0, out, q, runs_of(runs), rows, 100)
    nan = out.isnan().cpu()
    assert not nan[:80].any() and not nan[:90, 2:].any()
    assert nan[80:, :2, :32].all() and not nan[80:, :2, 32:].any() and nan[90:, 2:].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("shift", [0, 1])
def test_attention_rows_of_wider_tensors(dtype, rows, shift):
    """q a slice of a qkv row, out a slice of another tensor, of any alignment."""
    c = make([rows + 90], 2, 64)
    fill(c, [rows + 90])
    wide_q = randn(rows, 8 * 64 + 3 * shift, seed=5).to(dtype)
    wide_o = torch.full((rows, 6 * 64 + 5 * shift), 3, dtype=dtype, device="cuda")
    q, out = (w[:, shift:shift + 256].unflatten(1, (4, 64)) for w in (wide_q, wide_o))
    runs = [(0, rows, 0, 90)]
    c.attention(0, out, q, runs_of(runs), rows, rows + 90)
    check_attention(c, 0, q, out, runs, 2)
    assert (wide_o[:, :shift] == 3).all() and (wide_o[:, shift + 256:] == 3).all()


def test_attention_of_runs_outside_their_range():
    """Bad sequences and pages: zeros or the positions that exist, a bit set, nothing else touched."""
    lib = _lib.load()
    for rows in (1, 20):
        c = make([100, 30], 1, 64, layers=1)
        fill(c, [100, 30])
        q = randn(40, 2, 64, seed=1)
        for run in ((0, rows, 2, 0), (0, rows, -1, 5), (40, rows, 0, 0), (-rows, rows, 0, 0), (0, rows, 0, 200)):
            out = torch.full_like(q, 3)
            c.attention(0, out, q, runs_of([run]), rows, 100)
            torch.cuda.synchronize()
            assert lib.cats_gpu_device_error() == 0x40, run
            assert (out[rows:] == 3).all()
            if run[0]:
                assert (out == 3).all()
            elif run[2]:
                assert (out[:rows] == 0).all()
            lib.cats_gpu_clear_device_error()
        out = torch.full_like(q, 3)                              # a hole in the table: its 64 positions are left out
        c.table[0, 0] = -1
        c.attention(0, out, q, runs_of([(0, rows, 0, 100 - rows)]), rows, 100)
        assert torch.isfinite(out).all() and lib.cats_gpu_device_error() == 0x40
        lib.cats_gpu_clear_device_error()


@pytest.mark.parametrize("hints", [(1, 1), (0, 0), (3000, 100000)])
@pytest.mark.parametrize("new,lens", [([1, 1], [900, 70]), ([90, 20], [300, 20])])
def test_attention_hints(hints, new, lens):
    """max_rows and max_len size the launch only."""
    c = make(lens, 1, 64)
    fill(c, lens)
    q, out, runs = attend(c, 0, new, lens, 2, torch.float32, hints=hints)
    check_attention(c, 0, q, out, runs, 2, untouched=3)


def test_attention_is_the_same_every_time():
    for dtype in TYPES:
        for new, lens in (([1] * 5, [3000, 17, 900, 64, 2048]), ([200, 9], [700, 300])):
            c = make(lens, 2, 128, layers=1)
            fill(c, lens)
            got = [attend(c, 0, new, lens, 4, dtype)[1] for _ in range(3)]
            assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_long_cache_offsets():
    """A pool past 4 GiB: pages at its far end are read and written where they are."""
    n_kv, hs, layers = 8, 128, 80                                # 5.9 MB a page
    pages = 900                                                  # 5.3 GB
    c = kv.Cache.empty(pages, layers, n_kv, hs, 1, 3)
    c.table.copy_(torch.tensor([[899, 0, 898]], dtype=torch.int32))
    x = randn(150, n_kv, hs, seed=1)
    c.append(79, x, x * 2, runs_of([(0, 150, 0, 0)]), 150)
    k, v = torch.empty_like(x), torch.empty_like(x)
    c.read(79, k, v, runs_of([(0, 150, 0, 0)]), 150)
    assert np.array_equal(k.double().cpu().numpy(), blocks(x.double().cpu().numpy()))
    q, out, runs = attend(c, 79, [1], [150], 1, torch.float32, extra=0)
    kd, vd = k.double().cpu().numpy(), v.double().cpu().numpy()
    s = np.einsum("hd,lhd->hl", q[0].double().cpu().numpy(), kd) / math.sqrt(hs)
    p = np.exp(s - s.max(1, keepdims=True))
    want = np.einsum("hl,lhd->hd", p / p.sum(1, keepdims=True), vd)
    assert np.abs(out[0].double().cpu().numpy() - want).max() < 1e-5 * np.abs(vd).max()
    c.copy_pages([899, 898], [3, 897])
    assert torch.equal(c.pool[899], c.pool[3]) and torch.equal(c.pool[898], c.pool[897])
    del c


# -------------------------------------------------------------- page copies
@pytest.mark.parametrize("hs,n_kv,layers,pages,moves", [(32, 1, 1, 2, 1), (64, 3, 2, 90, 40), (128, 8, 4, 30, 15),
                                                        (32, 1, 1, 5000, 2400)])
def test_copy_pages(hs, n_kv, layers, pages, moves):
    g = torch.Generator().manual_seed(moves)
    pool = torch.randint(0, 256, (pages, layers, n_kv, 72 * hs), generator=g, dtype=torch.uint8)
    c = kv.Cache(pool.cuda(), torch.full((1, 1), -1, dtype=torch.int32, device="cuda"))
    order = torch.randperm(pages, generator=g)
    src = order[torch.randint(0, moves, (moves,), generator=g)].tolist()      # a source may serve several copies
    dst = order[moves:2 * moves].tolist()
    c.copy_pages(src, dst)
    pool[dst] = pool[src]
    assert torch.equal(c.pool.cpu(), pool)
    for bad in (([src[0]], [src[0]]), ([src[0]], [pages]), ([0, 0], [1, 1])):
        with pytest.raises(_lib.CatsGpuError):
            c.copy_pages(*bad)
    assert torch.equal(c.pool.cpu(), pool)


# ------------------------------------------------------------------ together
def test_a_conversation():
    """Prompt, fork, decode both branches with copy-on-write, drop one,
    compact: the rows of the cache and the attention over it stay those of
    plain sequences."""
    n_kv, mul, hs, max_pages = 2, 2, 64, 8
    r = random.Random(1)
    pages = kv.Pages(20, 4, max_pages)
    c = kv.Cache.empty(20, 1, n_kv, hs, 4, max_pages)
    c.pool.fill_(255)
    plain = {s: (np.zeros((0, n_kv, hs)), np.zeros((0, n_kv, hs))) for s in range(4)}
    step = [0]

    def add(seqs, ns):
        copies = [pages.write(s, plain[s][0].shape[0], n) for s, n in zip(seqs, ns)]
        for src, dst in copies:
            c.copy_pages(src, dst)
        c.table.copy_(torch.from_numpy(pages.table()))
        step[0] += 1
        k, v = (randn(sum(ns), n_kv, hs, seed=100 * step[0] + i) for i in (0, 1))
        q = randn(sum(ns), n_kv * mul, hs, seed=100 * step[0] + 2)
        first, runs = 0, []
        for s, n in zip(seqs, ns):
            runs.append((first, n, s, plain[s][0].shape[0]))
            plain[s] = tuple(np.concatenate([a, blocks(x[first:first + n].double().cpu().numpy())])
                             for a, x in zip(plain[s], (k, v)))
            first += n
        c.append(0, k, v, runs_of(runs), max(ns))
        out = torch.empty_like(q)
        c.attention(0, out, q, runs_of(runs), max(ns), max(plain[s][0].shape[0] for s in seqs))
        check_attention(c, 0, q, out, runs, mul)

    def same():
        for s, (k, v) in plain.items():
            if len(k):
                hk, hv = held(c, 0, s, len(k))
                assert np.array_equal(hk, k) and np.array_equal(hv, v)

    add([0, 1], [100, 30])
    pages.fork(0, 2, 100)
    plain[2] = plain[0]
    pages.fork(0, 3, 70)
    plain[3] = tuple(a[:70] for a in plain[0])
    for _ in range(4):
        add([0, 1, 2, 3], [1, 1, 1, 1])
    add([3], [60])
    same()
    pages.truncate(0, 0)
    plain[0] = (np.zeros((0, n_kv, hs)), np.zeros((0, n_kv, hs)))
    src, dst = pages.compact()
    c.copy_pages(src, dst)
    c.table.copy_(torch.from_numpy(pages.table()))
    same()
    add([1, 2, 3, 0], [r.randint(1, 40) for _ in range(4)])
    same()


def test_captured_and_replayed():
    """append, attention and page copies recorded into one graph and replayed on new data, on a stream of its own."""
    lens = [130, 65]
    c = make(lens, 1, 64, layers=1, spare=4)
    fill(c, lens)
    used = set(c.table.flatten().tolist())
    free = [p for p in range(c.n_pages) if p not in used]
    k, v, q = (randn(2, 1 if i < 2 else 4, 64, seed=i) for i in range(3))
    out = torch.zeros_like(q)
    run_list = [(0, 1, 0, 129), (1, 1, 1, 64)]
    runs = runs_of(run_list)
    src, dst = [int(c.table[0, 0])], [free[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        c.append(0, k, v, runs, 1, stream=s.cuda_stream)
        c.attention(0, out, q, runs, 1, 130, stream=s.cuda_stream)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            c.append(0, k, v, runs, 1, stream=s.cuda_stream)
            c.attention(0, out, q, runs, 1, 130, stream=s.cuda_stream)
            c.copy_pages(src, dst, stream=s.cuda_stream)
    for seed in (7, 8):
        for i, t in enumerate((k, v, q)):
            t.copy_(randn(*t.shape, seed=seed * 10 + i))
        c.pool[dst] = 0
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_attention(c, 0, q, out, run_list, 4)
        assert np.array_equal(held(c, 0, 0, 130)[0][129:], blocks(k[:1].double().cpu().numpy()))
        assert torch.equal(c.pool[dst], c.pool[src])


def test_tensors_that_do_not_fit_are_refused():
    c = make([64], 2, 64)
    x = randn(4, 2, 64)
    run = runs_of([(0, 4, 0, 0)])
    q = randn(4, 4, 64)
    bad = [lambda: c.append(0, x.double(), x.double(), run, 4), lambda: c.append(0, x[:, :1], x[:, :1], run, 4),
           lambda: c.append(0, x, x[:3], run, 4), lambda: c.append(0, x, x.half(), run, 4),
           lambda: c.append(0, x.cpu(), x.cpu(), run, 4), lambda: c.append(0, x, x, run.cpu(), 4),
           lambda: c.append(0, x, x, run.long(), 4), lambda: c.append(0, x, x, run[:, :3], 4),
           lambda: c.append(2, x, x, run, 4), lambda: c.append(0, x.transpose(1, 2).contiguous().transpose(1, 2), x, run, 4),
           lambda: c.append(0, x[:1].expand(4, 2, 64), x, run, 4), lambda: c.attention(0, q, q[:, :3], run, 4, 4),
           lambda: c.attention(0, q[:3], q, run, 4, 4), lambda: c.attention(0, q.half(), q, run, 4, 4),
           lambda: c.copy_pages([0], [0, 1]), lambda: kv.Cache(c.pool[..., :100], c.table),
           lambda: kv.Cache(c.pool.float(), c.table), lambda: kv.Cache(c.pool, c.table.long()),
           lambda: kv.Cache(c.pool.cpu(), c.table.cpu())]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError, _lib.CatsGpuError)):
            f()
            pytest.fail(str(i))
