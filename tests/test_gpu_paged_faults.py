"""Failure detection of the many-row attention kernel's bounded waits (about 2 s of SM clocks), without
a GPU fault: SQ_TEST_WITHHOLD_PIECE=2 makes the process's second launch leave one thread block without
word of its first piece. Every wait of that block runs out, the block returns, and the next status
check reports a timeout."""
import os
import time

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _child(q, kind):
    os.environ["SQ_TEST_WITHHOLD_PIECE"] = "2"
    try:
        from sqb200 import lib, paged
        from test_gpu_paged import KINDS, Setup, dev
        s = Setup(31, 2, 64, 64, [300], [6000])  # a few row tiles, each cut between many thread blocks
        x = dev(s.rows(8 * 64, kind, 1.5)).to(KINDS[kind])
        first = paged.attention(s.dcache, s.batch, x)  # launch 1
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        paged.status()
        t0 = time.monotonic()
        out = paged.attention(s.dcache, s.batch, x)  # launch 2
        torch.cuda.synchronize()
        try:
            paged.status()
            got = "none"
        except lib.KernelError as e:
            got = e.kind
        took = time.monotonic() - t0
        same = []
        fresh = paged.PagedBatch(s.batch.q_start, s.batch.kv_len, s.batch.page_table, 300, 300)
        for length in (2500, 6000):  # the same batch and workspace; row tiles cut into fewer parts, then as many as before
            s.batch.kv_len.fill_(length)
            out.zero_()
            paged.attention(s.dcache, s.batch, x, out=out)
            same.append(bool(torch.equal(out, paged.attention(s.dcache, fresh, x))))
            torch.cuda.synchronize()
            paged.status()
        with torch.cuda.graph(graph):
            paged.attention(s.dcache, s.batch, x, out=out)
        graph.replay()
        torch.cuda.synchronize()
        paged.status()
        q.put((got, took, same + [bool(torch.equal(out, first))]))
    except Exception as e:  # report instead of hanging the parent
        q.put((repr(e), 0.0, []))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_an_expired_wait_is_reported_and_the_batch_stays_usable(gpu_lib, kind):
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_child, args=(q, kind))
    p.start()
    try:
        got, took, same = q.get(timeout=300)
    finally:
        p.join(timeout=120)
        if p.is_alive():
            p.kill()
    assert got == "Timeout", got
    assert 0.5 < took < 60, took
    assert same == [True] * 3
