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
import weakref

import torch

from . import lib
from .lib import KernelError, _check

_KINDS = {torch.float32: lib.F32, torch.bfloat16: lib.BF16}
_SHAPE, _TYPE, _ARG = 1, 2, 5
_INT_MAX = 2**31 - 1


def _need(ok, code, what):
    if not ok:
        raise KernelError(code, what)


def _kind(t):
    kind = _KINDS.get(t.dtype)
    if kind is None:
        raise KernelError(_TYPE, "rows must be float32 or bfloat16")
    return kind


def _rows(t, rows, width, dtype, device, what):
    """Address and row stride of a [rows, width] tensor of dtype on the device whose rows may be
    a slice of wider ones."""
    if t.dtype is not dtype:
        raise KernelError(_TYPE, f"{what}: {dtype} is wanted")
    if t.shape != (rows, width):
        raise KernelError(_SHAPE, f"{what}: {rows} rows of {width} elements are wanted")
    stride, step = t.stride()
    if step != 1 and width > 1:
        raise KernelError(_SHAPE, f"{what}: a row's elements must be consecutive")
    if t.get_device() != device:
        raise KernelError(_ARG, f"{what}: a CUDA tensor of the current device is wanted")
    return t.data_ptr(), stride if rows > 1 else width  # one row: its stride says nothing


def _device_of(cache, batch):
    """The current device, which has to be the cache's and the batch's."""
    device = _device()
    if cache.device != device or batch.device != device:
        raise KernelError(_ARG, "cache and batch have to be on the current CUDA device")
    return device


# The smallest calls take a few microseconds of GPU time, so the binding spends as little as
# it can: entry points are looked up once, structs are passed by address, streams come from
# torch's raw lookup, and tensors that this module makes itself are not checked again.
_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch.cuda.current_device


_entries = {}


def _bind(name):
    """The library's entry point `name`: structs are passed as addresses. The interpreter lock is
    given up meanwhile: a status copy, or a launch into a full queue, waits for the GPU
    (0.1 us a call: append_one's two calls 19.6 with the lock kept, 19.75 us)."""
    lib.load()
    f = getattr(C.CDLL(lib.LIB_PATH), name)
    f.restype, types = lib.SIGNATURES[name]
    f.argtypes = [C.c_void_p if issubclass(t, C._Pointer) else t for t in types]
    _entries[name] = f
    return f


def _fn(name):
    return _entries.get(name) or _bind(name)


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
        self.device = k.get_device()
        self.n_pages, self.n_kv_heads, self.page, self.head_dim = k.shape
        self.shape_key = (self.n_kv_heads, self.page, self.head_dim)
        self.row, self.half, self.scale = self.n_kv_heads * self.head_dim, self.head_dim // 2, self.head_dim ** -0.5
        self.like = {t: torch.empty(0, dtype=t, device=k.device) for t in _KINDS}  # for new tensors of these types
        self.desc = lib.PagedCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        self.ref = C.addressof(self.desc)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, page=64, device="cuda"):
        codes = [torch.full((n_pages, n_kv_heads, page, head_dim), 128, dtype=torch.uint8, device=device)
                 for _ in range(2)]
        return cls(*codes, *(torch.zeros((n_pages, n_kv_heads), device=device) for _ in range(2)))


_batches = weakref.WeakSet()  # those that hold a workspace


class PagedBatch:
    """One step: sequence b has rows q_start[b] .. q_start[b + 1] - 1 of the step's tensors,
    the last of the kv_len[b] positions that it holds with them; page_table [n_seqs,
    pages_per_seq] names its pages (entries past kv_len, and with a window
    those of pages that no new token sees, are not read). The arrays are int32
    CUDA tensors and are read by the kernels: their contents may change between calls, with
    n_tokens rows in all and at most max_new of one sequence. The
    attention's workspace is kept here from the first call on, so calls with one batch must be
    ordered on the device (a graph captured before any other call gets workspaces of its own)."""

    def __init__(self, q_start, kv_len, page_table, n_tokens, max_new):
        for t in (q_start, kv_len, page_table):
            _need(t.dtype == torch.int32, _TYPE, "batch arrays are int32")
            _need(t.is_contiguous(), _SHAPE, "batch arrays are contiguous")
            _need(t.is_cuda and t.device == q_start.device, _ARG, "batch arrays are CUDA tensors of one device")
        _need(page_table.dim() == 2 and kv_len.shape == page_table.shape[:1] and
              q_start.shape == (kv_len.shape[0] + 1,), _SHAPE,
              "q_start [n_seqs + 1], kv_len [n_seqs], page_table [n_seqs, pages_per_seq]")
        self.q_start, self.kv_len, self.page_table, self.device = q_start, kv_len, page_table, q_start.get_device()
        self.n_seqs, self.n_tokens, self.max_new = kv_len.shape[0], n_tokens, max_new
        self.desc = lib.PagedBatchDesc(q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(), self.n_seqs,
                                       n_tokens, max_new, page_table.shape[1])
        self.ref = C.addressof(self.desc)
        self._workspaces = {}

    def workspace(self, cache, n_heads, stream=None):
        """(tensor, address, bytes, raw stream it was made on) for attention over caches of this
        shape, on the current stream (whose raw value may be given)."""
        if stream is None:
            stream = _raw_stream(_device())
        key = (cache.shape_key, n_heads)
        ws = self._workspaces.get(key)
        if ws is None:
            size = C.c_size_t()
            _check(lib.load().sq_paged_attention_workspace(C.pointer(cache.desc), C.pointer(self.desc), n_heads,
                                                           C.byref(size)))
            t = torch.zeros(size.value, dtype=torch.uint8, device=cache.k.device)
            ws = (t, t.data_ptr(), size.value, stream)
            if not torch.cuda.is_current_stream_capturing():  # zeros that a graph writes are its own calls' alone
                self._workspaces[key] = ws
                _batches.add(self)
        elif ws[3] != stream and not torch.cuda.is_current_stream_capturing():
            ws[0].record_stream(torch.cuda.current_stream())  # the memory outlives the batch until that stream is done
        return ws


def append(cache, batch, k, v, cos, sin, q=None, q_out=None):
    """Rotate k [n_tokens, n_kv_heads * head_dim] to its positions and store it and v in the
    pages; rotate q [n_tokens, n_heads * head_dim], if given, and return it (in q_out, which
    may be q, or a new tensor). cos, sin: [positions, head_dim / 2] float32."""
    n, width, dtype, device = batch.n_tokens, cache.row, k.dtype, _device_of(cache, batch)
    kind = _kind(k)
    kp, ks = _rows(k, n, width, dtype, device, "k")
    vp, vs = _rows(v, n, width, dtype, device, "v")
    positions = cos.shape[0]
    for t in (cos, sin):
        if (t.shape != (positions, cache.half) or t.dtype is not torch.float32 or not t.is_contiguous() or
                t.get_device() != device):
            raise KernelError(_SHAPE, "rotation tables are contiguous float32 [positions, head_dim / 2] on the GPU")
    qp = qop = None
    qs = qos = n_heads = 0
    if q is not None:
        q_width = q.shape[1] if q.dim() == 2 else 0
        n_heads = q_width // cache.head_dim
        if n_heads * cache.head_dim != q_width or not n_heads:
            raise KernelError(_SHAPE, "q: rows of whole heads are wanted")
        qp, qs = _rows(q, n, q_width, dtype, device, "q")
        if q_out is None:
            q_out = torch.empty_like(q)
            qop, qos = q_out.data_ptr(), q_width
        else:
            qop, qos = _rows(q_out, n, q_width, dtype, device, "q_out")
    st = _fn("sq_paged_append")(_raw_stream(device), cache.ref, batch.ref, kind, kp, ks, vp, vs, cos.data_ptr(),
                                sin.data_ptr(), positions, qp, qs, n_heads, qop, qos)
    if st:
        _check(st)
    return q_out


def attention(cache, batch, q, window=0, sinks=0, scale=None, out=None):
    """Causal grouped attention of q [n_tokens, n_heads * head_dim] over the cache: the query
    at position p sees the positions <= p, with window > 0 only the last `window` of them
    and the first `sinks` ones. scale: head_dim ** -0.5 unless given."""
    n, dtype, device = batch.n_tokens, q.dtype, _device_of(cache, batch)
    width = q.shape[1] if q.dim() == 2 else 0
    n_heads = width // cache.head_dim
    if n_heads * cache.head_dim != width or not n_heads:
        raise KernelError(_SHAPE, "q: rows of whole heads are wanted")
    kind = _kind(q)
    qp, qs = _rows(q, n, width, dtype, device, "q")
    if out is None:
        out = torch.empty_like(q)
        op, os_ = out.data_ptr(), width
    else:
        op, os_ = _rows(out, n, width, dtype, device, "out")
    if window > _INT_MAX or sinks > _INT_MAX:
        window, sinks = min(window, _INT_MAX), min(sinks, _INT_MAX)
    stream = _raw_stream(device)
    held, ws, ws_bytes, _ = batch.workspace(cache, n_heads, stream)
    st = _fn("sq_paged_attention")(stream, cache.ref, batch.ref, kind, qp, qs, n_heads,
                                   cache.scale if scale is None else scale, window, sinks, op, os_, ws, ws_bytes)
    if st:
        _check(st)
    return out


def read(cache, batch, first, count, dtype=torch.float32):
    """The values of `count` positions of each sequence from first[b] (int32 CUDA tensor) on:
    k, v [n_seqs, count, n_kv_heads * head_dim], zeros past kv_len[b]."""
    n, device = batch.n_seqs, _device_of(cache, batch)
    if (first.shape != (n,) or first.dtype is not torch.int32 or first.get_device() != device or
            not first.is_contiguous()):
        raise KernelError(_SHAPE, "first: one int32 position of each sequence on the GPU")
    if not 0 <= count <= _INT_MAX:
        raise KernelError(_SHAPE, "count: 0 to 2^31 - 1 positions")
    kind = _KINDS.get(dtype)
    if kind is None:
        raise KernelError(_TYPE, "values are read as float32 or bfloat16")
    k = cache.like[dtype].new_empty((n, count, cache.row))
    v = torch.empty_like(k)
    st = _fn("sq_paged_read")(_raw_stream(device), cache.ref, batch.ref, first.data_ptr(), count, kind,
                              k.data_ptr(), v.data_ptr())
    if st:
        _check(st)
    return k, v


def status(clear=True):
    """sq_paged_status: raise what the kernels found wrong in a batch's arrays (call after
    synchronizing). After a Timeout the device's workspaces are made as new: a block that
    gave up leaves its counters short."""
    try:
        _check(_fn("sq_paged_status")(int(clear)))
    except KernelError as e:
        if e.kind == "Timeout":
            for batch in list(_batches):
                for t, *_ in batch._workspaces.values():
                    if t.device.index == _device():
                        t.zero_()
            torch.cuda.current_stream().synchronize()  # before calls on any stream
        raise
