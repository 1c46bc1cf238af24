"""The paged 8-bit key/value cache over the C ABI (include/squirrel_cuda.h): rotation and
append, attention, reading back. No counterpart in the reference, whose cache is one f32
sequence (models/common/kv_cache.rs:8-78).

    cache = PagedCache.empty(n_pages, n_kv_heads, head_dim, page=64)      # one a layer
    batch = PagedBatch(q_start, kv_len, page_table, n_tokens, max_new)    # one a step
    q = append(cache, batch, k, v, cos, sin, q=q)
    out = attention(cache, batch, q)

Tensors live on the current CUDA device and calls run on torch's current stream. Errors
raise lib.KernelError. What only the kernels can see in a batch's arrays (a page id
outside the cache, a length beyond the page table, ...) is recorded on the device:
status() raises it after a synchronization.
"""
import ctypes as C

import torch

from . import lib
from .lib import KernelError, _check, _stream

_KINDS = {torch.float32: lib.F32, torch.bfloat16: lib.BF16}
_SHAPE, _TYPE, _ARG = 1, 2, 5


def _need(ok, code, what):
    if not ok:
        raise KernelError(code, what)


def _kind(t):
    kind = _KINDS.get(t.dtype)
    _need(kind is not None, _TYPE, "rows must be float32 or bfloat16")
    return kind


def _rows(t, rows, width, dtype, what):
    """A [rows, width] tensor of dtype whose rows may be a slice of wider ones."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != width or (width > 1 and t.stride(1) != 1):
        raise KernelError(_SHAPE, f"{what}: {rows} rows of {width} consecutive elements are wanted")
    if t.dtype != dtype:
        raise KernelError(_TYPE, f"{what}: {dtype} is wanted")
    if not t.is_cuda:
        raise KernelError(_ARG, f"{what}: a CUDA tensor is wanted")
    return t.data_ptr(), t.stride(0)


class PagedCache:
    """One layer's pages: codes k, v [n_pages, n_kv_heads, page, head_dim] uint8 (value =
    (code - 128) * scale) and scales [n_pages, n_kv_heads] float32."""

    def __init__(self, k, v, k_scale, v_scale):
        for t in (k, v):
            _need(t.dim() == 4 and t.shape == k.shape and t.is_contiguous(), _SHAPE,
                  "codes are contiguous [n_pages, n_kv_heads, page, head_dim]")
            _need(t.dtype == torch.uint8, _TYPE, "codes are uint8")
        for t in (k_scale, v_scale):
            _need(t.shape == k.shape[:2] and t.is_contiguous(), _SHAPE, "scales are contiguous [n_pages, n_kv_heads]")
            _need(t.dtype == torch.float32, _TYPE, "scales are float32")
        _need(all(t.is_cuda and t.device == k.device for t in (k, v, k_scale, v_scale)), _ARG,
              "a cache is CUDA tensors of one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page, self.head_dim = k.shape
        self.desc = lib.PagedCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        self.ref = C.pointer(self.desc)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, page=64, device="cuda"):
        codes = [torch.full((n_pages, n_kv_heads, page, head_dim), 128, dtype=torch.uint8, device=device)
                 for _ in range(2)]
        return cls(*codes, *(torch.zeros((n_pages, n_kv_heads), device=device) for _ in range(2)))


class PagedBatch:
    """One step: sequence b has rows q_start[b] .. q_start[b + 1] - 1 of the step's tensors,
    the last of the kv_len[b] positions that it holds with them; page_table [n_seqs,
    pages_per_seq] names its pages (entries past kv_len are not read). The arrays are int32
    CUDA tensors and are read by the kernels: their contents may change between calls
    within what n_tokens (rows in all) and max_new (most of one sequence) say. The
    attention's workspace is kept here, so calls with one batch must be ordered on the
    device."""

    def __init__(self, q_start, kv_len, page_table, n_tokens, max_new):
        for t in (q_start, kv_len, page_table):
            _need(t.dtype == torch.int32, _TYPE, "batch arrays are int32")
            _need(t.is_contiguous(), _SHAPE, "batch arrays are contiguous")
            _need(t.is_cuda, _ARG, "batch arrays are CUDA tensors")
        _need(page_table.dim() == 2 and kv_len.shape == page_table.shape[:1] and
              q_start.shape == (kv_len.shape[0] + 1,), _SHAPE,
              "q_start [n_seqs + 1], kv_len [n_seqs], page_table [n_seqs, pages_per_seq]")
        self.q_start, self.kv_len, self.page_table = q_start, kv_len, page_table
        self.n_tokens, self.max_new = n_tokens, max_new
        self.desc = lib.PagedBatchDesc(q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(), kv_len.shape[0],
                                       n_tokens, max_new, page_table.shape[1])
        self.ref = C.pointer(self.desc)
        self._workspaces = {}

    def workspace(self, cache, n_heads):
        key = (n_heads, cache.n_kv_heads, cache.head_dim, cache.page)
        ws = self._workspaces.get(key)
        if ws is None:
            size = C.c_size_t()
            _check(lib.load().sq_paged_attention_workspace(cache.ref, self.ref, n_heads, C.byref(size)))
            t = torch.zeros(size.value, dtype=torch.uint8, device=cache.k.device)
            ws = self._workspaces[key] = (t, t.data_ptr(), size.value)
        return ws


def append(cache, batch, k, v, cos, sin, q=None, q_out=None):
    """Rotate k [n_tokens, n_kv_heads * head_dim] to its positions and store it and v in the
    pages; rotate q [n_tokens, n_heads * head_dim], if given, and return it (in q_out, which
    may be q, or a new tensor). cos, sin: [positions, head_dim / 2] float32."""
    width = cache.n_kv_heads * cache.head_dim
    kind = _kind(k)
    kp, ks = _rows(k, batch.n_tokens, width, k.dtype, "k")
    vp, vs = _rows(v, batch.n_tokens, width, k.dtype, "v")
    for t in (cos, sin):
        _need(t.dim() == 2 and t.shape[1] == cache.head_dim // 2 and t.shape[0] == cos.shape[0] and
              t.is_contiguous() and t.dtype == torch.float32 and t.is_cuda, _SHAPE,
              "rotation tables are contiguous float32 [positions, head_dim / 2] on the GPU")
    qp = qop = None
    qs = qos = n_heads = 0
    if q is not None:
        _need(q.dim() == 2 and q.shape[1] % cache.head_dim == 0, _SHAPE, "q: rows of whole heads are wanted")
        n_heads = q.shape[1] // cache.head_dim
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qp, qs = _rows(q, batch.n_tokens, q.shape[1], k.dtype, "q")
        qop, qos = _rows(q_out, batch.n_tokens, q.shape[1], k.dtype, "q_out")
    _check(lib.load().sq_paged_append(_stream(), cache.ref, batch.ref, kind, kp, ks, vp, vs, cos.data_ptr(),
                                      sin.data_ptr(), cos.shape[0], qp, qs, n_heads, qop, qos))
    return q_out


def attention(cache, batch, q, window=0, sinks=0, scale=None, out=None):
    """Causal grouped attention of q [n_tokens, n_heads * head_dim] over the cache: the query
    at position p sees the positions <= p, with window > 0 only the last `window` of them
    and the first `sinks` ones. scale: head_dim ** -0.5 unless given."""
    _need(q.dim() == 2 and q.shape[1] % cache.head_dim == 0, _SHAPE, "q: rows of whole heads are wanted")
    n_heads = q.shape[1] // cache.head_dim
    kind = _kind(q)
    qp, qs = _rows(q, batch.n_tokens, q.shape[1], q.dtype, "q")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    op, os_ = _rows(out, batch.n_tokens, q.shape[1], q.dtype, "out")
    _, ws, ws_bytes = batch.workspace(cache, n_heads)
    _check(lib.load().sq_paged_attention(_stream(), cache.ref, batch.ref, kind, qp, qs, n_heads,
                                         cache.head_dim ** -0.5 if scale is None else scale, window, sinks, op, os_,
                                         ws, ws_bytes))
    return out


def read(cache, batch, first, count, dtype=torch.float32):
    """The values of `count` positions of each sequence from first[b] (int32 CUDA tensor) on:
    k, v [n_seqs, count, n_kv_heads * head_dim], zeros past kv_len[b]."""
    n = batch.kv_len.shape[0]
    _need(first.shape == (n,) and first.dtype == torch.int32 and first.is_cuda and first.is_contiguous(), _SHAPE,
          "first: one int32 position of each sequence on the GPU")
    _need(dtype in _KINDS, _TYPE, "values are read as float32 or bfloat16")
    shape = (n, count, cache.n_kv_heads * cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.k.device)
    v = torch.empty(shape, dtype=dtype, device=cache.k.device)
    _check(lib.load().sq_paged_read(_stream(), cache.ref, batch.ref, first.data_ptr(), count, _KINDS[dtype],
                                    k.data_ptr(), v.data_ptr()))
    return k, v


def status(clear=True):
    """sq_paged_status: raise what the kernels found wrong in a batch's arrays (call after
    synchronizing)."""
    _check(lib.load().sq_paged_status(int(clear)))
