"""The paged attention at the edges of what its arguments and batches may say, against tests/paged_oracle.py."""
import numpy as np
import pytest

import paged_oracle as P
from test_gpu_paged import KINDS, Setup, as_kind, dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_short_prompts_leave_the_second_row_tile_idle(gpu_lib, hd, kind):
    """Row tiles of up to 128 rows and one or two key blocks, some of more rows between them: a thread block goes
    through several of them while one of its product warps has nothing to do. The result, and equal bits on every call."""
    from sqb200 import paged
    news = [20 + i % 12 if i % 7 else 33 + i for i in range(300)]
    s = Setup(21, 8, hd, 32, news, [n + (i * 11) % 60 for i, n in enumerate(news)])
    q = s.rows(32 * hd, kind, 1.5)
    first = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]))
    for _ in range(100):
        assert torch.equal(paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind])), first)
    s.check_attention(32, kind, q=q)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("sinks", [0, 3])
@pytest.mark.parametrize("window", [255, 256, 257, 2**30, 2**31 - 16, 2**31 - 1, 2**31 + 5, 2**40])
def test_windows_as_long_as_the_table_and_longer(gpu_lib, window, sinks, kind):
    """A window that holds every position there can be hides nothing, whatever its size. (The table here has 16
    pages of 16: the oracle takes the window as it is.)"""
    for heads, news, lens in ((8, [1, 3], [1, 9]), (8, [40, 90, 1, 2], [40, 100, 240, 2])):
        Setup(22, 2, 64, 16, news, lens).check_attention(heads, kind, window=window, sinks=sinks)


BIG = [  # news, lens: rows of the one kernel, of the other, of both
    [1, 2], [300, 190],
    [200, 90], [420, 300],
    [150, 1], [400, 260],
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ratio", [1e6, 1e10, 1e20])
@pytest.mark.parametrize("where", [0, 3, 10])
@pytest.mark.parametrize("news,lens", list(zip(BIG[0::2], BIG[1::2])), ids=str)
def test_values_beside_far_larger_ones_without_weight(gpu_lib, news, lens, where, ratio, hd, kind):
    """One page has V scales `ratio` times the others', and keys that every query scores about 290 octaves below the
    others: the result is that of the small values alone, to the bound that goes by the largest of those."""
    from sqb200 import paged
    s = Setup(23, 2, hd, 16, news, lens)
    s.cache["vs"] /= np.float32(ratio)
    for b, n in enumerate(lens):
        s.cache["vs"][s.table[b, where]] *= np.float32(ratio)
        s.cache["k"][s.table[b, where]] = 1  # -127 in every dimension
        s.cache["ks"][s.table[b, where]] = 0.05
    for n, t in (("k", s.dcache.k), ("ks", s.dcache.k_scale), ("vs", s.dcache.v_scale)):
        t.copy_(dev(s.cache[n]))
    q = np.full((sum(news), 8 * hd), 4, np.float32)
    got = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]))
    torch.cuda.synchronize()
    paged.status()
    want, size = P.attention(s.cache, s.q_start, lens, s.table, q, 8)
    # what the far larger page adds is below 2^-200 of the rest; every row sees another page before or after it
    size[..., 1] = 127 * 1.5 / 60 / ratio
    seen = np.concatenate([(np.arange(n - k, n) >= 16) | (where > 0) for k, n in zip(news, lens)])
    over = np.abs(got.float().cpu().numpy().reshape(want.shape) - want) / (P.bound(want, size, kind))
    assert over[seen].max() <= 1


@pytest.mark.parametrize("what", ["begins_late", "ends_early", "none"])
@pytest.mark.parametrize("news", [[1, 2, 1], [40, 40, 40]], ids=str)
def test_rows_of_no_sequence_are_recorded(gpu_lib, news, what):
    """q_start has to run from 0 to n_tokens: rows outside it would be left as they were."""
    from sqb200 import lib, paged
    s = Setup(24, 2, 64, 16, news, [50, 90, 60])
    q_start = s.batch.q_start.clone()
    if what == "begins_late":
        q_start[0] = 1
    elif what == "ends_early":
        q_start[3] -= 1
    else:
        q_start[:] = 0
    batch = paged.PagedBatch(q_start, s.batch.kv_len, s.batch.page_table, sum(news), max(news))
    q, k = dev(s.rows(512, "f32")), dev(s.rows(128, "f32"))
    cos, sin = (dev(x) for x in P.rotation(128, 64))
    paged.status()
    for call in (lambda: paged.attention(s.dcache, batch, q), lambda: paged.append(s.dcache, batch, k, k, cos, sin, q=q),
                 lambda: paged.read(s.dcache, batch, dev(np.int32([0, 0, 0])), 90)):
        call()
        torch.cuda.synchronize()
        with pytest.raises(lib.KernelError) as e:
            paged.status()
        assert e.value.kind == "InvalidArgument" and "q_start" in str(e.value)
        paged.status()  # cleared


def test_a_batch_first_used_in_a_capture(gpu_lib):
    """The captured call must not leave the batch a workspace that only its replay fills with zeros."""
    from sqb200 import paged
    s = Setup(25, 2, 64, 64, [1, 1], [9000, 7000])
    q = s.rows(512, "f32")
    x = dev(q)
    other = paged.PagedBatch(s.batch.q_start, s.batch.kv_len, s.batch.page_table, 2, 1)
    want = paged.attention(s.dcache, other, x)
    torch.cuda.synchronize()
    dirty, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(dirty):  # memory that later captures in the same pool are given
        torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    dirty.replay()
    with torch.cuda.graph(graph, pool=dirty.pool()):
        out = paged.attention(s.dcache, s.batch, x)
    torch.cuda.synchronize()
    assert torch.equal(paged.attention(s.dcache, s.batch, x), want)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(paged.attention(s.dcache, s.batch, x), want)


@pytest.mark.parametrize("hd,news,n_seqs,pages", [(32, 2048, 4500, 256), (64, 16384, 900, 512)], ids=str)
def test_sequences_that_claim_the_same_rows_are_recorded(gpu_lib, hd, news, n_seqs, pages):
    """Every other sequence claims all rows and very many keys: together more (row tile, key tile) pairs than 32 bits
    count. Nothing is looked for beyond the last sequence, the call is recorded, and the device is as usable as before."""
    from sqb200 import lib, paged
    s = Setup(26, 8, hd, 256, [1], [1])
    q_start = np.int32([0, news] * (n_seqs // 2) + [0])
    table = np.full((n_seqs, pages), s.table[0, 0], np.int32)
    batch = paged.PagedBatch(dev(q_start), dev(np.full(n_seqs, 256 * pages, np.int32)), dev(table), news, news)
    q = torch.randn(news, 32 * hd, device="cuda")
    paged.status()
    paged.attention(s.dcache, batch, q)
    torch.cuda.synchronize()
    with pytest.raises(lib.KernelError) as e:
        paged.status()
    assert "q_start" in str(e.value)
    paged.status()
    Setup(26, 2, hd, 16, [1, 40, 1], [50, 90, 20]).check_attention(8, "f32")


def test_far_more_rows_than_positions(gpu_lib):
    """A sequence of 2^22 new tokens and 100 positions: all but the last rows stand before position 0. Counted as if
    they had keys, the row tiles' key blocks would not fit 32 bits."""
    from sqb200 import paged
    n, lens = 1 << 22, 100
    s = Setup(27, 8, 64, 64, [lens], [lens])
    tail = as_kind(s.rows(512, "bf16"), "bf16")
    q = torch.full((n, 512), 3.0, dtype=torch.bfloat16, device="cuda")
    q[-lens:] = dev(tail).bfloat16()
    batch = paged.PagedBatch(dev(np.int32([0, n])), s.batch.kv_len, s.batch.page_table, n, n)
    out = paged.attention(s.dcache, batch, q)
    torch.cuda.synchronize()
    paged.status()
    assert not out[:-lens].any()
    want, size = P.attention(s.cache, [0, lens], [lens], s.table, tail, 8)
    over = np.abs(out[-lens:].float().cpu().numpy().reshape(want.shape) - want) / P.bound(want, size, "bf16")
    assert over.max() <= 1


def test_counters_past_32_bits(gpu_lib):
    """Many sequences beside one of many new tokens: more row tiles in the workspace than 32 bits count, and the last
    sequence's, which are cut between thread blocks, at its far end."""
    from sqb200 import paged
    n_seqs, news, last, lens = 65535, 4200 * 64, 300, 1000
    s = Setup(28, 8, 64, 64, [last], [lens])
    q_start = np.full(n_seqs + 1, news, np.int32)
    q_start[0], q_start[-1] = 0, news + last
    kv_len = np.zeros(n_seqs, np.int32)
    kv_len[-1] = lens
    table = np.full((n_seqs, s.table.shape[1]), -1, np.int32)
    table[-1] = s.table[0]
    batch = paged.PagedBatch(dev(q_start), dev(kv_len), dev(table), news + last, news)
    tail = as_kind(s.rows(2048, "bf16", 1.5), "bf16")
    q = torch.zeros(news + last, 2048, dtype=torch.bfloat16, device="cuda")
    q[news:] = dev(tail).bfloat16()
    assert batch.workspace(s.dcache, 32)[2] > 4 << 31
    for _ in range(2):
        out = paged.attention(s.dcache, batch, q)
        torch.cuda.synchronize()
        paged.status()
        want, size = P.attention(s.cache, [0, last], [lens], s.table, tail, 32)
        over = np.abs(out[news:].float().cpu().numpy().reshape(want.shape) - want) / P.bound(want, size, "bf16")
        assert over.max() <= 1 and not out[:news].any()


def test_the_workspace_outlives_its_batch_on_other_streams(gpu_lib):
    """A call on another stream than the workspace's, which is still to run when the batch goes: its memory is not given
    to the first stream's next tensor."""
    from sqb200 import paged
    s = Setup(29, 2, 64, 64, [1, 1], [9000, 7000])
    x = dev(s.rows(512, "f32"))
    want = paged.attention(s.dcache, s.batch, x)
    size = s.batch.workspace(s.dcache, 8)[2]
    torch.cuda.synchronize()
    for _ in range(3):
        batch = paged.PagedBatch(s.batch.q_start, s.batch.kv_len, s.batch.page_table, 2, 1)
        paged.attention(s.dcache, batch, x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)  # some 50 ms
            out = paged.attention(s.dcache, batch, x)
        del batch
        other = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255)
        side.synchronize()
        assert torch.equal(out, want)
        del other


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("news", [3, 100])
@pytest.mark.parametrize("power", [-120, -60, 14, 16, 18, 20, 24, 34, 90, 114, 118, 120])
def test_query_rows_of_any_size(gpu_lib, power, news, kind):
    """Rows of 2^power in one dimension, K scales of 2^-7: scores of about 2^(power - 3). Large rows leave the key with the
    largest code there all the weight, tiny ones weight all keys alike."""
    from sqb200 import paged
    s = Setup(30, 2, 64, 16, [news], [200])
    s.cache["ks"][:] = 2.0**-7
    s.cache["k"][:, :, :, 5] = 100 + s.rng.integers(0, 2, s.cache["k"].shape[:3])
    best = s.rng.integers(0, 200 - news, 2)
    for g in range(2):
        s.cache["k"][s.table[0, best[g] // 16], g, best[g] % 16, 5] = 102
    for n, t in (("k", s.dcache.k), ("ks", s.dcache.k_scale)):
        t.copy_(dev(s.cache[n]))
    q = np.zeros((news, 8, 64), np.float32)
    q[:, :, 5] = 2.0**power
    got = paged.attention(s.dcache, s.batch, dev(q.reshape(news, 512)).to(KINDS[kind])).float().cpu().numpy()
    paged.status()
    want, size = P.attention(s.cache, s.q_start, s.lens, s.table, q.reshape(news, 512), 8)
    if power > 0:
        size[..., 0] = 0  # the other keys' weights are below 2^-20: an error of scores moves nothing
    over = np.abs(got.reshape(q.shape) - want) / P.bound(want, size, kind)
    assert over.max() <= 1
