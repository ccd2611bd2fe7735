"""Paged KV cache in Q4_0 blocks over libcatsgpu (cats_gpu_kv_*).

`Cache` wraps two torch CUDA tensors, the pool of pages and the page table, and
runs the operators on them: append, read, attention, copy_pages.  `Pages` is
the host's bookkeeping: which page holds which tokens of which sequence.

A batch is a CUDA int32 tensor of runs [n][4]: first row, rows, sequence,
position of the first row.  stream: a cudaStream_t, or None for torch's current
one (the legacy default: the library's own, which is ordered with it).  A
call is asynchronous on its stream: what else works on its tensors on another
is the caller's to order.  Their memory is kept until the call is done with it.
No gradient passes through the cache: rows that want one are refused.
"""
import ctypes as C
from array import array

import numpy as np

from . import _lib

PAGE = 64
F32, F16, BF16 = 0, 1, 30
_TYPES = {}


def page_bytes(n_layers, n_kv_heads, head_size):
    """Bytes of one page of the pool."""
    n = _lib.load().cats_gpu_kv_page_bytes(n_layers, n_kv_heads, head_size)
    if not n:
        raise ValueError(f"no cache of {n_layers} layers, {n_kv_heads} heads of {head_size}: "
                         "head_size is a multiple of 32 up to 128")
    return n


def _type(t):
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    got = _TYPES.get(t.dtype)
    if got is None:
        raise TypeError(f"float32, float16 or bfloat16 is wanted, not {t.dtype}")
    return got


def _ints(x):
    """(address, length, owner) of host integers as C ints."""
    if isinstance(x, (list, tuple)):   # a third of the time through numpy
        a = array("i", x)
        return a.buffer_info()[0], len(a), a
    a = np.asarray(x)
    if a.ndim != 1:
        raise ValueError("a list of integers is wanted")
    if a.size and a.dtype.kind not in "iu":
        raise TypeError(f"integers are wanted, not {a.dtype}")
    if a.size and not -2**31 <= int(a.min()) <= int(a.max()) < 2**31:
        raise OverflowError("page numbers of 32 bits are wanted")
    a = np.ascontiguousarray(a, np.int32)
    return a.ctypes.data, a.size, a


def _int32(*values):
    """Refuse what C's int would wrap."""
    for x in values:
        if not -2**31 <= x < 2**31:
            raise OverflowError(f"{x} does not fit 32 bits")


def _rows(t, heads, hs, device, what):
    """Row stride of a tensor [rows][heads][hs] whose rows are whole."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != hs:
        raise ValueError(f"{what}: shape [rows, {heads}, {hs}] is wanted, not {list(shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the cache on {device}")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and hs > 1) or (s1 != hs and heads > 1):
        raise ValueError(f"{what}: the values of a row must be contiguous")
    if t.requires_grad:
        _lib.no_gradient(what)
    width = heads * hs
    if shape[0] <= 1:
        return width
    if s0 < width:
        raise ValueError(f"{what}: rows overlap")
    return s0


class Cache:
    """pool: uint8 [n_pages, n_layers, n_kv_heads, 72 * head_size]; table: int32
    [n_seqs, max_pages], -1 where a sequence has no page.  Both are the
    caller's; the operators read the table's current contents."""

    def __init__(self, pool, table):
        import torch
        if pool.dtype != torch.uint8 or pool.dim() != 4 or not pool.is_contiguous() or pool.shape[3] % 2304:
            raise ValueError("pool: a contiguous uint8 tensor [pages, layers, kv heads, 72 * head_size] is wanted")
        if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
            raise ValueError("table: a contiguous int32 tensor [sequences, pages] is wanted")
        if not pool.is_cuda or table.device != pool.device:
            raise ValueError("pool and table must be on the same CUDA device")
        self._lib = _lib.check_device(pool.device)
        self.pool, self.table, self._dev, self._i32 = pool, table, pool.device, torch.int32
        self.n_pages, self.n_layers, self.n_kv_heads = pool.shape[:3]
        self.head_size = pool.shape[3] // 72
        self._c = _lib.KvC(pool.data_ptr(), table.data_ptr(), *pool.shape[:3], self.head_size, *table.shape)
        self._p = C.addressof(self._c)

    @classmethod
    def empty(cls, n_pages, n_layers, n_kv_heads, head_size, n_seqs, max_pages, device="cuda"):
        """A cache of its own tensors, no sequence holding a page."""
        import torch
        per = page_bytes(1, 1, head_size)
        return cls(torch.empty(n_pages, n_layers, n_kv_heads, per, dtype=torch.uint8, device=device),
                   torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device))

    def _batch(self, runs):
        shape = runs.shape
        if len(shape) != 2 or shape[1] != 4 or not runs.is_contiguous() or runs.dtype != self._i32:
            raise ValueError("runs: a contiguous int32 tensor [n, 4] is wanted")
        if runs.device != self._dev:
            raise ValueError(f"runs are on {runs.device}, the cache on {self._dev}")
        return runs.data_ptr(), shape[0]

    def _on(self, stream, *tensors):
        if stream is None:
            return _lib.current_stream(self._dev.index)
        _lib.other_stream(self._dev, stream, (self.pool, self.table, *tensors))
        return stream

    def _kv(self, fn, layer, k, v, runs, max_rows, stream):
        dev = self._dev
        ld_k = _rows(k, self.n_kv_heads, self.head_size, dev, "k")
        ld_v = _rows(v, self.n_kv_heads, self.head_size, dev, "v")
        if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
            raise ValueError("k and v must have the same type and rows")
        batch, stream = self._batch(runs), self._on(stream, k, v, runs)
        _lib.check(fn(self._p, layer, k.data_ptr(), v.data_ptr(), _type(k), ld_k, ld_v, k.shape[0], *batch, max_rows,
                      stream), "kv")

    def append(self, layer, k, v, runs, max_rows, stream=None):
        """Quantize rows k, v [rows, n_kv_heads, head_size] into the pages of `layer`."""
        self._kv(self._lib.cats_gpu_kv_append_dev, layer, k, v, runs, max_rows, stream)

    def read(self, layer, k, v, runs, max_rows, stream=None):
        """The values the cache holds for the runs' positions, into k and v."""
        self._kv(self._lib.cats_gpu_kv_read_dev, layer, k, v, runs, max_rows, stream)
        return k, v

    def attention(self, layer, out, q, runs, max_rows, max_len, stream=None):
        """out[row] = causal attention of q[row] over its sequence; q and out
        [rows, n_heads, head_size].  max_rows: the longest run; max_len: the
        largest position + 1."""
        heads = q.shape[1] if q.dim() == 3 else 0
        if heads == 0 or heads % self.n_kv_heads:
            raise ValueError(f"q: [rows, heads, head_size] with heads a multiple of {self.n_kv_heads} is wanted")
        dev = self._dev
        ld_q = _rows(q, heads, self.head_size, dev, "q")
        ld_o = _rows(out, heads, self.head_size, dev, "out")
        if q.dtype != out.dtype or q.shape[0] != out.shape[0]:
            raise ValueError("q and out must have the same type and rows")
        batch, stream = self._batch(runs), self._on(stream, q, out, runs)
        _lib.check(self._lib.cats_gpu_kv_attention_dev(self._p, layer, out.data_ptr(), q.data_ptr(), _type(q), heads,
                                                       ld_o, ld_q, q.shape[0], *batch, max_rows, max_len, stream),
                   "kv attention")
        return out

    def copy_pages(self, src, dst, stream=None):
        """Pages dst[i] = pages src[i] (host integers); no page may be written
        twice, nor both read and written."""
        (src, n, _a), (dst, m, _b) = _ints(src), _ints(dst)
        if n != m:
            raise ValueError("src and dst must be lists of the same length")
        _lib.check(self._lib.cats_gpu_kv_copy_pages_dev(self._p, src, dst, n, self._on(stream)), "copy_pages")


class Pages:
    """Which page of a cache holds which tokens of which sequence (host only)."""

    def __init__(self, n_pages, n_seqs, max_pages):
        _int32(n_pages, n_seqs, max_pages)
        self._lib = _lib.load()
        self._shape = (n_seqs, max_pages)
        self.n_pages = n_pages
        self._h = self._lib.cats_gpu_kv_pages_create(n_pages, n_seqs, max_pages)
        if not self._h:
            _lib.check(None, "kv_pages_create")
            raise _lib.CatsGpuError("kv_pages_create failed")

    def _copies(self, room, call, what):
        src, dst, n = np.zeros(room, np.int32), np.zeros(room, np.int32), C.c_int()
        _lib.check(call(C.c_void_p(src.ctypes.data), C.c_void_p(dst.ctypes.data), C.byref(n)), what)
        return src[:n.value], dst[:n.value]

    def write(self, seq, pos, n):
        """Make n positions from pos writable; returns the page copies (src, dst) to make first."""
        _int32(seq, pos, n)
        return self._copies(max(n, 0) // PAGE + 2,
                            lambda s, d, c: self._lib.cats_gpu_kv_pages_write(self._h, seq, pos, n, s, d, c),
                            "kv_pages_write")

    def fork(self, src_seq, dst_seq, length):
        """dst_seq becomes the first `length` tokens of src_seq, sharing its pages."""
        _int32(src_seq, dst_seq, length)
        _lib.check(self._lib.cats_gpu_kv_pages_fork(self._h, src_seq, dst_seq, length), "kv_pages_fork")

    def truncate(self, seq, length):
        """Keep the first `length` tokens of a sequence (0: free it)."""
        _int32(seq, length)
        _lib.check(self._lib.cats_gpu_kv_pages_truncate(self._h, seq, length), "kv_pages_truncate")

    def compact(self):
        """Renumber the used pages to the front; returns the page copies (src, dst) to make."""
        return self._copies(self.n_pages, lambda s, d, c: self._lib.cats_gpu_kv_pages_compact(self._h, s, d, c),
                            "kv_pages_compact")

    def length(self, seq):
        _int32(seq)
        return self._lib.cats_gpu_kv_pages_length(self._h, seq)

    @property
    def free(self):
        return self._lib.cats_gpu_kv_pages_free(self._h)

    def table(self):
        """A copy of the page table, int32 [n_seqs, max_pages]."""
        p = C.cast(self._lib.cats_gpu_kv_pages_table(self._h), C.POINTER(C.c_int))
        return np.ctypeslib.as_array(p, shape=self._shape).copy()

    def __del__(self):
        if getattr(self, "_h", None):
            self._lib.cats_gpu_kv_pages_destroy(self._h)
            self._h = None
