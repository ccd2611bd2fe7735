"""Log probabilities of given tokens over libcatsgpu (cats_gpu_logprobs_dev)."""
from . import _lib
from .kv import _type

MAX_K = 32


def logprobs(logits, targets=None, k=0, entropy=True, stream=None):
    """Of the rows of logits [rows, vocab] (CUDA; float32, float16 or bfloat16;
    rows may be a wider tensor's): (log softmax at targets [rows] or None,
    entropy [rows] or None, ids of the k <= 32 likeliest [rows, k], their log
    probabilities [rows, k]).  A negative target gives 0; of equal logits the
    lower id comes first.  stream: a cudaStream_t, or None for the current one;
    the results are made on it, and whoever reads them on another waits for it.
    They carry no gradient: logits that want one are refused."""
    import torch
    if logits.requires_grad:
        _lib.no_gradient("logits")
    if logits.dim() != 2 or not logits.is_cuda or logits.shape[1] == 0 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: a CUDA tensor [rows, vocab] with contiguous rows is wanted")
    rows, vocab = logits.shape
    dev = logits.device
    lib = _lib.check_device(dev)
    ld = logits.stride(0) if rows > 1 else vocab
    if ld < vocab:
        raise ValueError("logits: rows overlap")
    if targets is not None and (targets.dtype != torch.int32 or targets.shape != (rows,) or targets.device != dev or
                                not targets.is_contiguous()):
        raise ValueError("targets: a contiguous int32 tensor [rows] on the logits' device is wanted")
    if not 0 <= k <= MAX_K:
        raise ValueError(f"k: 0 to {MAX_K} is wanted, not {k}")
    if stream is None:
        stream = _lib.current_stream(dev.index)
    else:
        other = _lib.other_stream(dev, stream, (logits, targets))
        if other is not None:   # the results' memory is that stream's
            with torch.cuda.stream(other):
                return _launch(lib, logits, targets, k, entropy, rows, vocab, ld, dev, stream)
    return _launch(lib, logits, targets, k, entropy, rows, vocab, ld, dev, stream)


def _launch(lib, logits, targets, k, entropy, rows, vocab, ld, dev, stream):
    import torch
    # (four tensors are made in less time than one is cut in three)
    f32 = torch.float32
    lp = torch.empty(rows, dtype=f32, device=dev) if targets is not None else None
    h = torch.empty(rows, dtype=f32, device=dev) if entropy else None
    ids = torch.empty(rows, k, dtype=torch.int32, device=dev)
    top = torch.empty(rows, k, dtype=f32, device=dev)
    _lib.check(lib.cats_gpu_logprobs_dev(
        logits.data_ptr(), _type(logits), rows, vocab, ld, targets.data_ptr() if targets is not None else None, k,
        lp.data_ptr() if lp is not None else None, h.data_ptr() if entropy else None, ids.data_ptr() if k else None,
        top.data_ptr() if k else None, stream), "logprobs")
    return lp, h, ids, top
