"""Refusals of the paged cache's and the verification's entry points: they come from the
host's checks, before any launch, so they need no GPU. Pointers are never touched."""
import ctypes as C

import pytest

OK_CACHE = dict(k=256, v=256, k_scale=256, v_scale=256, n_pages=4, n_kv_heads=2, page=16, head_dim=64)
OK_BATCH = dict(q_start=256, kv_len=256, page_table=256, n_seqs=2, n_tokens=3, max_new=2, pages_per_seq=4)


def structs(cache, batch):
    from sqb200 import lib
    return (C.byref(lib.PagedCacheDesc(**{**OK_CACHE, **cache})), C.byref(lib.PagedBatchDesc(**{**OK_BATCH, **batch})))


def append(cache={}, batch={}, dtype=0, k=256, ks=128, v=256, vs=128, cos=256, sin=256, rows=64, q=256, qs=512, heads=8,
           qo=256, qos=512):
    from sqb200 import lib
    c, b = structs(cache, batch)
    return lib.STATUS[lib.load().sq_paged_append(None, c, b, dtype, k, ks, v, vs, cos, sin, rows, q, qs, heads, qo, qos)]


def attention(cache={}, batch={}, dtype=0, q=256, qs=512, heads=8, scale=0.125, window=0, sinks=0, out=256, os=512, ws=256,
              ws_bytes=1 << 30):
    from sqb200 import lib
    c, b = structs(cache, batch)
    return lib.STATUS[lib.load().sq_paged_attention(None, c, b, dtype, q, qs, heads, scale, window, sinks, out, os, ws,
                                                    ws_bytes)]


def read(cache={}, batch={}, first=256, count=5, dtype=0, k=256, v=256):
    from sqb200 import lib
    c, b = structs(cache, batch)
    return lib.STATUS[lib.load().sq_paged_read(None, c, b, first, count, dtype, k, v)]


CALLS = [append, attention, read]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("cache,kind", [
    (dict(k=None), "InvalidArgument"), (dict(v_scale=None), "InvalidArgument"), (dict(n_pages=0), "ShapeMismatch"),
    (dict(n_kv_heads=-1), "ShapeMismatch"), (dict(page=24), "ShapeMismatch"), (dict(page=8), "ShapeMismatch"),
    (dict(page=512), "ShapeMismatch"), (dict(head_dim=96), "ShapeMismatch"), (dict(k=264), "TensorAlignmentError"),
    (dict(v_scale=258), "TensorAlignmentError")])
def test_cache_refusals(call, cache, kind):
    assert call(cache=cache) == kind


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("batch,kind", [
    (dict(q_start=None), "InvalidArgument"), (dict(page_table=None), "InvalidArgument"), (dict(n_seqs=0), "ShapeMismatch"),
    (dict(n_seqs=70000), "ShapeMismatch"), (dict(n_tokens=-1), "ShapeMismatch"), (dict(max_new=0), "ShapeMismatch"),
    (dict(max_new=4), "ShapeMismatch"), (dict(max_new=1), "ShapeMismatch"), (dict(pages_per_seq=0), "ShapeMismatch"),
    (dict(kv_len=255), "TensorAlignmentError")])
def test_batch_refusals(call, batch, kind):
    assert call(batch=batch) == kind


def test_append_refusals():
    assert append(dtype=8) == "InvalidType"
    assert append(k=None) == "InvalidArgument"
    assert append(v=None) == "InvalidArgument"
    assert append(cos=None) == "InvalidArgument"
    assert append(rows=0) == "ShapeMismatch"
    assert append(sin=260) == "TensorAlignmentError"
    assert append(ks=127) == "ShapeMismatch"      # rows overlap
    assert append(vs=130) == "TensorAlignmentError"
    assert append(dtype=30, ks=132) == "TensorAlignmentError"
    assert append(k=264) == "TensorAlignmentError"
    assert append(heads=0) == "ShapeMismatch"
    assert append(qs=508) == "ShapeMismatch"
    assert append(qo=None) == "InvalidArgument"
    assert append(batch=dict(n_tokens=0, max_new=0), k=None) == "Ok"  # nothing to append


def test_attention_refusals():
    assert attention(dtype=2) == "InvalidType"
    assert attention(heads=9) == "ShapeMismatch"
    assert attention(heads=0) == "ShapeMismatch"
    assert attention(window=-1) == "ShapeMismatch"
    assert attention(sinks=-1) == "ShapeMismatch"
    assert attention(q=None) == "InvalidArgument"
    assert attention(out=None) == "InvalidArgument"
    assert attention(os=514) == "TensorAlignmentError"
    assert attention(qs=511) == "ShapeMismatch"
    assert attention(out=260) == "TensorAlignmentError"
    assert attention(ws=None) == "InvalidArgument"
    assert attention(ws=384 + 16) == "TensorAlignmentError"
    assert attention(ws_bytes=0) == "InvalidArgument"
    assert attention(batch=dict(n_tokens=0, max_new=0), q=None) == "Ok"


def test_read_refusals():
    assert read(dtype=8) == "InvalidType"
    assert read(count=-1) == "ShapeMismatch"
    assert read(first=None) == "InvalidArgument"
    assert read(v=None) == "InvalidArgument"
    assert read(k=264) == "TensorAlignmentError"
    assert read(count=0, first=None) == "Ok"


def test_workspace_size():
    from sqb200 import lib
    L, size = lib.load(), C.c_size_t()
    c, b = structs({}, {})
    assert L.sq_paged_attention_workspace(c, b, 8, C.byref(size)) == 0 and size.value > 0
    assert L.sq_paged_attention_workspace(c, b, 8, None) == 5
    assert L.sq_paged_attention_workspace(c, b, 7, C.byref(size)) == 1


def verify(target=256, ts=100, draft=256, ds=100, tokens=256, n=None, u=256, seqs=2, k=3, vocab=100, acc=256, out=256):
    from sqb200 import lib
    return lib.STATUS[lib.load().sq_verify_drafts(None, target, ts, draft, ds, tokens, n, u, seqs, k, vocab, acc, out)]


def test_verify_refusals():
    assert verify(target=None) == "InvalidArgument"
    assert verify(tokens=None) == "InvalidArgument"
    assert verify(out=None) == "InvalidArgument"
    assert verify(vocab=0) == "ShapeMismatch"
    assert verify(seqs=-1) == "ShapeMismatch"
    assert verify(k=-1) == "ShapeMismatch"
    assert verify(ts=99) == "ShapeMismatch"
    assert verify(ds=99) == "ShapeMismatch"
    assert verify(target=258) == "TensorAlignmentError"
    assert verify(seqs=0) == "Ok"
    assert verify(seqs=0, draft=None, ds=0) == "Ok"


def test_python_checks():
    """The binding refuses tensors that are not what the entry points take."""
    torch = pytest.importorskip("torch")
    from sqb200 import paged
    from sqb200.lib import KernelError
    codes, scale = torch.zeros((4, 2, 16, 64), dtype=torch.uint8), torch.zeros((4, 2))
    for args, kind in (((codes, codes[:3], scale, scale), "ShapeMismatch"), ((codes, codes, scale, scale[:, :1]), "ShapeMismatch"),
                       ((codes.int(), codes.int(), scale, scale), "InvalidType"),
                       ((codes, codes, scale.double(), scale), "InvalidType"),
                       ((codes, codes, scale, scale), "InvalidArgument")):  # host tensors
        with pytest.raises(KernelError) as e:
            paged.PagedCache(*args)
        assert e.value.kind == kind
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(KernelError) as e:
        paged.PagedBatch(i.long(), i, i, 1, 1)
    assert e.value.kind == "InvalidType"
