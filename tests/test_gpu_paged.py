"""The paged 8-bit cache on the GPU against tests/paged_oracle.py: append (codes, scales and
rotated queries equal bit for bit), attention (bounds derived in paged_oracle.bound), reading
back, and what the kernels record about a batch they cannot use."""
import numpy as np
import pytest

import paged_oracle as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

KINDS = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def as_kind(x, kind):
    """numpy f32 rounded to the rows' type."""
    return torch.from_numpy(x).to(KINDS[kind]).float().numpy()


class Setup:
    """A random cache and ragged batch, on the host and on the device."""

    def __init__(self, seed, kvh, hd, page, news, lens, spare=2, garbage=True):
        from sqb200 import paged
        self.rng = rng = np.random.default_rng(seed)
        self.kvh, self.hd, self.page, self.news, self.lens = kvh, hd, page, list(news), list(lens)
        per = [max(1, -(-n // page)) for n in lens]
        n_pages = sum(per) + spare
        order = rng.permutation(n_pages)
        self.table = np.full((len(lens), max(per) + 1), -1, np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        shape = (n_pages, kvh, page, hd)
        # every code value, tails included: what lies past a sequence's end is never used
        self.cache = {"k": rng.integers(1, 256, shape).astype(np.uint8), "v": rng.integers(1, 256, shape).astype(np.uint8),
                      "ks": (rng.uniform(0.3, 1.5, shape[:2]) / 60).astype(np.float32),
                      "vs": (rng.uniform(0.3, 1.5, shape[:2]) / 60).astype(np.float32)}
        if garbage:  # pages of no sequence
            self.cache["ks"][order[at:]] = np.nan
            self.cache["vs"][order[at:]] = np.inf
        self.dcache = paged.PagedCache(*(dev(self.cache[n]) for n in ("k", "v", "ks", "vs")))
        self.batch = paged.PagedBatch(dev(self.q_start), dev(np.int32(lens)), dev(self.table), int(sum(news)),
                                      max(max(news), 0))

    def rows(self, width, kind, size=1.0):
        return as_kind((self.rng.standard_normal((sum(self.news), width)) * size).astype(np.float32), kind)

    def check_attention(self, heads, kind, q=None, **kw):
        from sqb200 import paged
        q = self.rows(heads * self.hd, kind, 1.5) if q is None else as_kind(q, kind)
        got = paged.attention(self.dcache, self.batch, dev(q).to(KINDS[kind]), **kw)
        torch.cuda.synchronize()
        paged.status()
        want, size = P.attention(self.cache, self.q_start, self.lens, self.table, q, heads, **kw)
        got = got.float().cpu().numpy().astype(np.float64).reshape(want.shape)
        over = np.abs(got - want) / P.bound(want, size, kind)
        assert np.isfinite(got).all() and over.max() <= 1, over.max()


# ---- append ------------------------------------------------------------------------

APPENDS = [  # kvh, hd, page, news, lens
    (8, 64, 64, [1], [1]),                       # the first token of all
    (8, 64, 64, [1], [1001]),
    (2, 32, 16, [1, 1, 1, 0], [16, 17, 48, 5]),  # a page's last, first and last again, an idle one
    (2, 64, 16, [5, 3, 0, 1, 7], [5, 20, 0, 33, 40]),
    (2, 128, 32, [70, 1, 33], [70, 64, 200]),
    (1, 256, 128, [129, 2], [130, 128]),
    (3, 64, 256, [300, 17], [600, 256]),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append_bit_exact(gpu_lib, case, kind):
    from sqb200 import paged
    kvh, hd, page, news, lens = case
    s = Setup(1, kvh, hd, page, news, lens)
    cos, sin = P.rotation(max(lens) + 3, hd)
    k, v, q = s.rows(kvh * hd, kind, 2.0), s.rows(kvh * hd, kind, 0.4), s.rows(3 * kvh * hd, kind)
    got = paged.append(s.dcache, s.batch, dev(k).to(KINDS[kind]), dev(v).to(KINDS[kind]), dev(cos), dev(sin),
                       q=dev(q).to(KINDS[kind]))
    torch.cuda.synchronize()
    paged.status()
    P.append(s.cache, s.q_start, lens, s.table, k, v, cos, sin)
    for name, t in (("k", s.dcache.k), ("v", s.dcache.v), ("ks", s.dcache.k_scale), ("vs", s.dcache.v_scale)):
        np.testing.assert_array_equal(t.cpu().numpy(), s.cache[name])
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(news, lens)]).astype(int)
    want = P.rotate(q.reshape(len(pos), -1, hd), cos[pos], sin[pos]).reshape(q.shape)
    np.testing.assert_array_equal(got.float().cpu().numpy(), as_kind(want, kind))


def test_append_token_by_token_raises_the_scale(gpu_lib):
    """Growing tokens raise the page's scale each time: the codes stay those of the restated
    steps, and every held value stays within half a step for each raise of its own step."""
    from sqb200 import paged
    s = Setup(2, 2, 32, 16, [1], [1], spare=0)
    rows = [np.float32(1.25)**i * s.rng.standard_normal((1, 64)).astype(np.float32) for i in range(16)]
    cos, sin = np.ones((16, 16), np.float32), np.zeros((16, 16), np.float32)
    for i, r in enumerate(rows):
        batch = paged.PagedBatch(dev(np.int32([0, 1])), dev(np.int32([i + 1])), s.batch.page_table, 1, 1)
        paged.append(s.dcache, batch, dev(r), dev(-r), dev(cos), dev(sin))
        P.append(s.cache, [0, 1], [i + 1], s.table, r, -r, cos, sin)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(s.dcache.k.cpu().numpy(), s.cache["k"])
    np.testing.assert_array_equal(s.dcache.v.cpu().numpy(), s.cache["v"])
    np.testing.assert_array_equal(s.dcache.k_scale.cpu().numpy(), s.cache["ks"])
    k, _ = paged.read(s.dcache, batch, dev(np.int32([0])), 16)
    step = s.cache["ks"][s.table[0, 0]].repeat(32)
    assert (np.abs(k.cpu().numpy()[0] - np.concatenate(rows)) <= 8.5 * step).all()  # 16 raises of half a step, and one


def test_append_special_values(gpu_lib):
    """NaN is stored as 0, infinities as the largest value, zeros and denormals as they are."""
    from sqb200 import paged
    s = Setup(3, 2, 32, 16, [4, 2, 3], [4, 2, 3])
    k, v = s.rows(64, "f32"), s.rows(64, "f32")
    k[0, 3], k[1, 5], k[2, 40], v[1, 0], v[2, 63] = np.nan, np.inf, -np.inf, np.nan, np.inf
    k[4:6], v[4:6] = 0, np.float32(3e-45)          # a page of zeros; one of the smallest denormal
    k[6:], v[6:] = np.inf, np.float32(3e38)         # nothing finite; the largest magnitudes
    cos, sin = np.ones((8, 16), np.float32), np.zeros((8, 16), np.float32)
    paged.append(s.dcache, s.batch, dev(k), dev(v), dev(cos), dev(sin))
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        P.append(s.cache, s.q_start, s.lens, s.table, k, v, cos, sin)
    for name, t in (("k", s.dcache.k), ("v", s.dcache.v), ("ks", s.dcache.k_scale), ("vs", s.dcache.v_scale)):
        np.testing.assert_array_equal(t.cpu().numpy(), s.cache[name])


def test_append_strided_rows_and_in_place(gpu_lib):
    """q, k and v as slices of one fused projection, q rotated in place, on another stream."""
    from sqb200 import paged
    s, ref = (Setup(4, 2, 64, 16, [3, 1, 9], [30, 16, 9]) for _ in range(2))
    rows = s.rows((8 + 2 + 2) * 64, "f32")
    cos, sin = P.rotation(32, 64)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = dev(rows)
        q, k, v = x[:, :512], x[:, 512:640], x[:, 640:]
        assert paged.append(s.dcache, s.batch, k, v, dev(cos), dev(sin), q=q, q_out=q) is q
    stream.synchronize()
    want_q = paged.append(ref.dcache, ref.batch, dev(rows[:, 512:640]), dev(rows[:, 640:]), dev(cos), dev(sin),
                          q=dev(rows[:, :512]))
    assert torch.equal(x[:, :512], want_q)
    np.testing.assert_array_equal(x[:, 512:].cpu().numpy(), rows[:, 512:])
    assert torch.equal(s.dcache.k, ref.dcache.k) and torch.equal(s.dcache.v, ref.dcache.v)


# ---- reading back ------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_read(gpu_lib, kind):
    from sqb200 import paged
    s = Setup(5, 3, 32, 16, [1, 1, 0], [37, 16, 5])
    first = [20, 10, -2]
    k, v = paged.read(s.dcache, s.batch, dev(np.int32(first)), 9, dtype=KINDS[kind])
    for got, codes, scales in ((k, "k", "ks"), (v, "v", "vs")):
        want = np.zeros((3, 9, 96), np.float32)
        for b in range(3):
            for i in range(9):
                p = first[b] + i
                if 0 <= p < s.lens[b]:
                    at = s.table[b, p // 16]
                    x = (s.cache[codes][at, :, p % 16].astype(np.float32) - 128) * s.cache[scales][at][:, None]
                    want[b, i] = x.reshape(-1)
        np.testing.assert_array_equal(got.float().cpu().numpy(), as_kind(want, kind))


# ---- attention ---------------------------------------------------------------------

ATTENTIONS = [  # heads, kvh, hd, page, news, lens
    (32, 8, 64, 64, [1], [1]),
    (32, 8, 64, 64, [1], [1001]),
    (8, 2, 32, 16, [1, 1, 1, 0, 1], [16, 17, 31, 40, 2]),
    (8, 2, 64, 16, [1, 1, 1], [65, 63, 129]),
    (16, 16, 64, 32, [1, 1], [100, 7]),             # every head its own keys
    (24, 8, 128, 16, [1, 1, 1], [33, 200, 64]),     # groups of 3
    (40, 8, 128, 64, [1, 2], [80, 333]),            # groups of 5
    (64, 8, 128, 128, [1], [300]),                  # groups of 8
    (8, 1, 256, 32, [1, 3], [77, 130]),             # one kv head, the widest head
    (36, 2, 32, 256, [1], [300]),                   # groups of 18
    (8, 2, 64, 16, [5, 3, 0, 1, 7], [5, 20, 0, 33, 40]),  # drafts; a sequence of new tokens only
    (8, 2, 128, 32, [17, 2], [100, 65]),
    (8, 2, 64, 64, [70, 1, 33], [70, 64, 200]),     # prompts among single tokens
    (8, 2, 128, 16, [130], [300]),
    (4, 4, 64, 64, [257], [513]),
    (8, 1, 256, 64, [40], [99]),
    (8, 2, 32, 64, [65], [120]),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", ATTENTIONS, ids=str)
def test_attention(gpu_lib, case, kind):
    heads, kvh, hd, page, news, lens = case
    Setup(6, kvh, hd, page, news, lens).check_attention(heads, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (16, 0), (40, 17), (64, 64), (100000, 3)])
@pytest.mark.parametrize("case", [(8, 2, 64, 16, [1, 3, 1, 0], [200, 65, 3, 9]), (8, 2, 128, 64, [150, 20], [400, 20]),
                                  (8, 2, 64, 64, [300], [700])], ids=str)
def test_attention_window(gpu_lib, case, window, sinks, kind):
    heads, kvh, hd, page, news, lens = case
    Setup(7, kvh, hd, page, news, lens).check_attention(heads, kind, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("news", [[18, 1, 7], [19, 8, 9, 1, 0, 18], [64, 8], [65, 9]], ids=str)
def test_attention_where_the_kernels_share_a_batch(gpu_lib, news, hd, kind):
    """Row counts on both sides of where sequences pass from the one kernel to the other (groups of 4)."""
    Setup(17, 2, hd, 32, news, [n + 61 * (i + 1) for i, n in enumerate(news)]).check_attention(8, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_pages_left_behind_by_the_window(gpu_lib, page, kind):
    """Pages that no new token sees may be gone: their entries and scales are not used."""
    news, lens, window, sinks = [1, 5, 90, 0], [500, 333, 700, 260], 70, 20
    s = Setup(16, 2, 64, page, news, lens)
    q = s.rows(8 * 64, kind, 1.5)
    want, size = P.attention(s.cache, s.q_start, lens, s.table, q, 8, window=window, sinks=sinks)
    for b, (new, n) in enumerate(zip(news, lens)):
        for p in range(-(-n // page)):
            if p * page >= sinks and (p + 1) * page - 1 <= n - new - window:
                for name in ("ks", "vs"):
                    s.cache[name][s.table[b, p]] = np.nan
                s.table[b, p] = -1
    assert (s.table[2, 3:] == -1).any()
    s.dcache.k_scale.copy_(dev(s.cache["ks"]))
    s.dcache.v_scale.copy_(dev(s.cache["vs"]))
    s.batch.page_table.copy_(dev(s.table))
    from sqb200 import paged
    got = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]), window=window, sinks=sinks)
    torch.cuda.synchronize()
    paged.status()
    over = np.abs(got.float().cpu().numpy().reshape(want.shape) - want) / P.bound(want, size, kind)
    assert over.max() <= 1


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("news,lens", [([4], [2]), ([1, 3], [0, 1]), ([90, 1], [40, 40])])
def test_attention_rows_that_see_nothing(gpu_lib, news, lens, kind):
    """More rows than positions: the first ones stand before position 0 and get zeros."""
    from sqb200 import paged
    s = Setup(8, 2, 64, 16, news, lens)
    q = s.rows(8 * 64, kind)
    out = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]))
    torch.cuda.synchronize()
    assert (out[:news[0] - lens[0]] == 0).all()
    s.check_attention(8, kind, q=q)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_score_ranges(gpu_lib, kind):
    """Scores that leave one key all the weight, equal scores, zero and tiny and huge rows, a
    negative and a zero scale, pages of zeros."""
    s = Setup(9, 2, 64, 16, [1] * 6, [50, 50, 50, 50, 33, 47])
    s.cache["ks"][s.table[2, 0]] = 0
    s.cache["vs"][s.table[2, :4]] = 0
    s.cache["vs"][s.table[4, 1]] = 1e-30
    s.cache["vs"][s.table[4, 2]] = 1e20
    for n, t in (("ks", s.dcache.k_scale), ("vs", s.dcache.v_scale)):
        t.copy_(dev(s.cache[n]))
    q = s.rows(8 * 64, kind)
    q[0] *= 40
    q[1] = 0
    q[3] = as_kind(q[3] * np.float32(1e-30), kind)
    q[5, 1:] = as_kind(q[5, 1:] * np.float32(2e-5), kind)  # one large element in the row's first head
    for scale in (None, 0.0, -0.3):
        s.check_attention(8, kind, q=q, **({} if scale is None else {"scale": scale}))


def test_attention_non_finite_rows_stay_alone(gpu_lib):
    """A query row with NaN or infinity spoils its own heads only."""
    from sqb200 import paged
    s = Setup(10, 2, 64, 16, [3, 80], [40, 90])
    q = s.rows(8 * 64, "f32")
    clean = paged.attention(s.dcache, s.batch, dev(q))
    q[1, 64 * 2 + 5], q[50, 0] = np.nan, np.inf
    got = paged.attention(s.dcache, s.batch, dev(q))
    torch.cuda.synchronize()
    bad = torch.zeros(83, 8, dtype=torch.bool)
    bad[1, 2] = bad[50, 0] = True
    got, clean = got.view(83, 8, 64).cpu(), clean.view(83, 8, 64).cpu()
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], clean[~bad])


def test_attention_strided_rows_streams_and_repeats(gpu_lib):
    """Slices of wider rows in and out, another stream, and equal bits on every call."""
    from sqb200 import paged
    s = Setup(11, 2, 64, 16, [1, 2, 30, 1], [700, 65, 90, 1500])
    q = s.rows(8 * 64, "f32")
    want = paged.attention(s.dcache, s.batch, dev(q))
    torch.cuda.synchronize()
    wide, out = torch.full((34, 768), 7.0, device="cuda"), torch.full((34, 640), -3.0, device="cuda")
    wide[:, 128:640] = dev(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            paged.attention(s.dcache, s.batch, wide[:, 128:640], out=out[:, 64:576])
    stream.synchronize()
    assert torch.equal(out[:, 64:576], want)
    assert (out[:, :64] == -3).all() and (out[:, 576:] == -3).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_long_prompts(gpu_lib, hd, kind):
    """Many row tiles, most of them cut between thread blocks: the result, and equal bits on every call
    (the products of a piece's last two key blocks are both done before its rows are written)."""
    from sqb200 import paged
    s = Setup(14, 8, hd, 64, [1100, 700], [1300, 700])
    q = s.rows(32 * hd, kind, 1.5)
    first = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]))
    for _ in range(20):
        assert torch.equal(paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind])), first)
    s.check_attention(32, kind, q=q)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_prompts_among_idle_sequences(gpu_lib, kind):
    """Short prompts far apart in a long batch: thread blocks finish their rows while the next prompt is looked for."""
    news, lens = [17 if b % 60 == 7 else 0 for b in range(6000)], [17 + b % 3 for b in range(6000)]
    Setup(15, 8, 64, 64, news, lens).check_attention(32, kind)


def test_attention_in_a_graph_follows_the_batch(gpu_lib):
    """A captured step replays with new lengths in the batch's arrays."""
    from sqb200 import paged
    s = Setup(12, 2, 64, 16, [1, 1], [600, 90])
    q = dev(s.rows(8 * 64, "f32"))
    out = paged.attention(s.dcache, s.batch, q)  # the workspace exists before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(s.dcache, s.batch, q, out=out)
    for lens in ([600, 90], [17, 1], [333, 64]):
        s.batch.kv_len.copy_(dev(np.int32(lens)))
        graph.replay()
        torch.cuda.synchronize()
        want, size = P.attention(s.cache, s.q_start, lens, s.table, q.cpu().numpy(), 8)
        over = np.abs(out.cpu().numpy().reshape(want.shape) - want) / P.bound(want, size, "f32")
        assert over.max() <= 1, over.max()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_offsets_past_32_bits(gpu_lib, kind):
    """A pool of more than 2^32 codes, the sequence's pages at its far end."""
    from sqb200 import paged
    hd, page, kvh = 128, 64, 8
    n_pages = (1 << 32) // (kvh * page * hd) + 24
    s = Setup(13, kvh, hd, page, [1, 70], [1001, 200], garbage=False)
    small = s.dcache
    big = paged.PagedCache(*(torch.empty((n_pages, kvh, page, hd), dtype=torch.uint8, device="cuda") for _ in range(2)),
                           *(torch.zeros((n_pages, kvh), device="cuda") for _ in range(2)))
    shift = n_pages - small.n_pages
    for n in ("k", "v", "k_scale", "v_scale"):
        getattr(big, n)[shift:] = getattr(small, n)
    table = s.batch.page_table.clone()
    table[table >= 0] += shift
    batch = paged.PagedBatch(s.batch.q_start, s.batch.kv_len, table, 71, 70)
    q, k = s.rows(32 * hd, kind), s.rows(kvh * hd, kind)
    cos, sin = P.rotation(1001, hd)
    for c, b in ((small, s.batch), (big, batch)):
        paged.append(c, b, dev(k).to(KINDS[kind]), dev(k).to(KINDS[kind]), dev(cos), dev(sin))
    assert torch.equal(big.k[shift:], small.k) and torch.equal(big.v_scale[shift:], small.v_scale)
    x = dev(q).to(KINDS[kind])
    assert torch.equal(paged.attention(big, batch, x), paged.attention(small, s.batch, x))
    first = dev(np.int32([950, 150]))
    for a, b in zip(paged.read(big, batch, first, 50), paged.read(small, s.batch, first, 50)):
        assert torch.equal(a, b)


# ---- what a batch's arrays may say -------------------------------------------------


@pytest.mark.parametrize("what", ["page", "page_negative", "length", "length_negative", "start", "max_new"])
def test_bad_batches_are_recorded_not_read_through(gpu_lib, what):
    from sqb200 import lib, paged
    s = Setup(14, 2, 64, 16, [1, 40, 1], [50, 90, 20])
    table, kv_len, q_start = s.batch.page_table.clone(), s.batch.kv_len.clone(), s.batch.q_start.clone()
    if what == "page":
        table[1, 4] = s.dcache.n_pages  # positions 64 to 79: read and written
    elif what == "page_negative":
        table[1, 4] = -7
    elif what == "length":
        kv_len[1] = 1 << 30
    elif what == "length_negative":
        kv_len[1] = -5
    elif what == "start":
        q_start[2] = 1 << 29
    max_new = 30 if what == "max_new" else 40
    batch = paged.PagedBatch(q_start, kv_len, table, 42, max_new)
    q, k = dev(s.rows(512, "f32")), dev(s.rows(128, "f32"))
    cos, sin = (dev(x) for x in P.rotation(128, 64))
    paged.status()
    for call in (lambda: paged.attention(s.dcache, batch, q), lambda: paged.append(s.dcache, batch, k, k, cos, sin, q=q),
                 lambda: paged.read(s.dcache, batch, dev(np.int32([0, 0, 0])), 90)):
        call()
        torch.cuda.synchronize()
        with pytest.raises(lib.KernelError) as e:
            paged.status()
        assert e.value.kind == "InvalidArgument"
        paged.status()  # cleared
    # the device is as usable as before
    s2 = Setup(14, 2, 64, 16, [1, 40, 1], [50, 90, 20])
    s2.check_attention(8, "f32")


def test_append_positions_outside_the_table_are_recorded(gpu_lib):
    from sqb200 import lib, paged
    s = Setup(15, 2, 64, 16, [1, 4], [50, 20])
    k = dev(s.rows(128, "f32"))
    before = s.dcache.k.clone()
    cos, sin = (dev(x) for x in P.rotation(18, 64))
    paged.append(s.dcache, s.batch, k, k, cos, sin)
    torch.cuda.synchronize()
    with pytest.raises(lib.KernelError) as e:
        paged.status()
    assert "rotation table" in str(e.value)
    page, last = s.table[1, 1], s.table[0, 3]
    assert torch.equal(s.dcache.k[last], before[last])                  # position 49: not written
    assert not torch.equal(s.dcache.k[page, :, :2], before[page, :, :2])  # 16 and 17 are
    assert torch.equal(s.dcache.k[page, :, 2:], before[page, :, 2:])      # 18 and 19 are not
