"""Speculative decoding over the C ABI: verification of drafted tokens from given random
numbers. No counterpart in the reference, whose generation takes one greedy token a step
(text_generator.rs:38-101)."""
import torch

from .lib import KernelError, _check
from .paged import _device, _fn, _raw_stream

_SHAPE, _TYPE, _ARG = 1, 2, 5


def _array(t, shape, dtype, device, what):
    if t.shape != shape or not t.is_contiguous():
        raise KernelError(_SHAPE, f"{what}: a contiguous {shape} tensor is wanted")
    if t.dtype is not dtype:
        raise KernelError(_TYPE, f"{what}: {dtype} is wanted")
    if t.get_device() != device:
        raise KernelError(_ARG, f"{what}: a CUDA tensor of the current device is wanted")
    return t.data_ptr()


def _probs(t, n, rows, vocab, device, what):
    """Address and row stride of [n, rows, vocab] float32 whose rows lie one stride apart (a slice
    of wider rows or of more of them). Broadcast or overlapping rows are refused: the kernel
    would read past the end of them."""
    if t.shape != (n, rows, vocab):
        raise KernelError(_SHAPE, f"{what}: [{n}, {rows}, {vocab}] is wanted")
    far, stride, step = t.stride()
    if rows == 1:
        stride = far  # the stride of a single row says nothing: rows are a sequence apart
    if n * rows < 2:
        stride = vocab
    elif vocab and (stride < vocab or (n > 1 and far != rows * stride)):
        raise KernelError(_SHAPE, f"{what}: [{n}, {rows}, {vocab}] with one stride between rows is wanted")
    if step != 1 and vocab > 1 and n * rows:
        raise KernelError(_SHAPE, f"{what}: a row's elements must be consecutive")
    if t.dtype is not torch.float32:
        raise KernelError(_TYPE, f"{what}: probabilities are float32")
    if t.get_device() != device:
        raise KernelError(_ARG, f"{what}: a CUDA tensor of the current device is wanted")
    return t.data_ptr(), stride


def verify_drafts(target, draft, tokens, uniform, n_draft=None):
    """target [n, K + 1, vocab]: the target's probabilities at each drafted token and after
    the last; draft [n, K, vocab]: the drafting distribution, or None when it was certain of
    its tokens; tokens [n, K] int32; uniform [n, K + 1] in [0, 1); n_draft [n] int32: tokens
    drafted for each sequence (None: K). Returns (accepted [n], tokens [n, K + 1]) int32:
    the accepted drafts, the token drawn after them, then -1."""
    if tokens.dim() != 2 or target.dim() != 3:
        raise KernelError(_SHAPE, "tokens are [n, K], target is [n, K + 1, vocab]")
    n, k = tokens.shape
    vocab, device = target.shape[2], _device()
    tp, ts = _probs(target, n, k + 1, vocab, device, "target")
    dp, ds = _probs(draft, n, k, vocab, device, "draft") if draft is not None else (None, 0)
    accepted, out = tokens.new_empty(n), tokens.new_empty((n, k + 1))
    st = _fn("sq_verify_drafts")(
        _raw_stream(device), tp, ts, dp, ds, _array(tokens, (n, k), torch.int32, device, "tokens"),
        _array(n_draft, (n,), torch.int32, device, "n_draft") if n_draft is not None else None,
        _array(uniform, (n, k + 1), torch.float32, device, "uniform"), n, k, vocab, accepted.data_ptr(), out.data_ptr())
    if st:
        _check(st)
    return accepted, out
