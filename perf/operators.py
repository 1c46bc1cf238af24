"""Serving operators of the paged 8-bit key/value cache: the measured cases.

Three operators, as one step of a batched server with drafted tokens uses them:

  append     rotate new queries and keys to their positions, quantize the keys and
             values into the pages of an 8-bit cache (one scale per page and head, raised
             when a new token needs it) and read the written pages back
  attention  causal grouped attention of the new tokens over that cache, optionally with
             a sliding window and a few first positions that stay visible
  verify     accept or reject drafted tokens against the target's probabilities and draw
             the next token, from given random numbers

`run` computes them in plain torch operations (own = False) or through sqb200.paged and
sqb200.speculative (own = True). The cache holds biased codes: value = (code - 128) * scale.
"""
import math
import sys

import torch

own = False

DEV = "cuda"
FRACTION_BITS = 38  # fixed-point bits of a probability's weight in the token draw
UNIFORM_BITS = 24   # bits of a uniform number in [0, 1) that count


def listed():
    def append(name, **kw):
        return dict(name=name, op="append", **kw)

    def attention(name, window=0, sinks=0, **kw):
        return dict(name=name, op="attention", window=window, sinks=sinks, **kw)

    small = dict(heads=32, kv_heads=8, head_dim=64)   # the 1B model's attention
    large = dict(heads=32, kv_heads=8, head_dim=128)  # the 8B model's attention
    return [
        # one chat on one GPU writes one token of one layer: latency
        append("append_one", type="f32", page=64, seqs=1, new=1, longest=1001, **small),
        # a server's decode step of a full batch, small pages
        append("append_batch", type="bf16", page=16, seqs=64, new=1, longest=8000, **large),
        # long prompts enter the cache
        append("append_prompt", type="f32", page=64, seqs=3, new=8192, longest=8231, **small),
        # one chat reads a short context: latency
        attention("attend_one", type="f32", page=64, seqs=1, new=1, longest=1001, **small),
        # a server's decode step over a ragged batch
        attention("attend_batch", type="bf16", page=16, seqs=64, new=1, longest=4000, **large),
        # few documents at the models' full context length
        attention("attend_long", type="f32", page=64, seqs=4, new=1, longest=131072, **small),
        # drafted tokens are scored together, a ragged number in each sequence
        attention("attend_drafts", type="f32", page=32, seqs=16, new=5, longest=4099, **small),
        # long chats under a sliding window with the first tokens kept
        attention("attend_window", type="bf16", page=64, seqs=32, new=1, longest=30000, window=1024, sinks=4, **large),
        # the second chunk of a prompt attends to the first and to itself
        attention("attend_chunk", type="f32", page=64, seqs=1, new=2048, longest=4133, **small),
        # two prompts of different lengths are prefilled behind cached prefixes
        attention("attend_prompts", type="bf16", page=64, seqs=2, new=4096, longest=8000, **large),
        # one chat checks four drafted tokens over the models' vocabulary: latency
        dict(name="verify_one", op="verify", seqs=1, drafts=4, vocab=128256, draft_probs=True),
        # a full batch checks its drafts
        dict(name="verify_batch", op="verify", seqs=64, drafts=5, vocab=128256, draft_probs=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "verify"])
    if op == "verify":
        vocab = _log(rng, 500, 160000)
        drafts = rng.randint(1, 8)
        return dict(op=op, seqs=min(64, max(1, _log(rng, 1, 64 * 6 * 128256 // (vocab * (drafts + 1))))), drafts=drafts,
                    vocab=vocab, draft_probs=rng.random() < 0.75)
    heads, kv_heads, head_dim = rng.choice(
        [(32, 8, 64), (32, 8, 64), (32, 8, 128), (32, 8, 128), (8, 2, 64), (8, 2, 32), (16, 16, 64), (24, 8, 128),
         (64, 8, 128), (8, 1, 256)])
    c = dict(op=op, type=rng.choice(["f32", "bf16"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             page=rng.choice([16, 32, 64, 128]))
    row = kv_heads * head_dim
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 8192), _log(rng, 9, 8192)])
        most = 2 * 8192 * 512 * 5 // (row + heads * head_dim)  # rows of the largest listed call and less
        new = min(new, most)
        seqs = _log(rng, 1, max(1, min(64, most // new)))
        longest = new + _log(rng, 1, 131072 // (seqs if new == 1 else 16)) - 1
        return dict(c, seqs=seqs, new=new, longest=longest)
    longest = _log(rng, 1, 131072)
    seqs = _log(rng, 1, max(1, min(64, 2 * 131072 * 512 // (longest * row))))
    mode = rng.choice(["one", "one", "few", "many"])
    room = 2 * 32 * 2048 * 128 * min(4000, longest) // (heads * head_dim * longest * seqs)  # inside the largest listed
    new = min(longest, 1 if mode == "one" else _log(rng, 2, 8) if mode == "few" else _log(rng, 9, 4096), max(1, room))
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    return dict(c, seqs=seqs, new=new, longest=longest, window=window, sinks=rng.choice([0, 4, 33]) if window else 0)


# ---- sizes that follow from a case -------------------------------------------------


def new_tokens(c):
    """New tokens of each sequence: ragged; in a larger batch the last one is idle."""
    n = [max(1, c["new"] - (i * 37) % (c["new"] // 2 + 1)) for i in range(c["seqs"])]
    if c["seqs"] > 3:
        n[-1] = 0
    return n


def lengths(c):
    """Positions of each sequence after the step: from a quarter of the longest up to it."""
    n = c["seqs"]
    return [max(k, c["longest"] - (3 * c["longest"] * ((i * 29) % n)) // (4 * n)) for i, k in enumerate(new_tokens(c))]


def _first_pages(c):
    """Start of the page that each sequence's first new token falls in."""
    return [(length - n) // c["page"] * c["page"] for length, n in zip(lengths(c), new_tokens(c))]


def _visible(c, pos):
    """Number of cached positions the query at `pos` sees."""
    if not c["window"] or pos < c["window"]:
        return pos + 1
    return c["window"] + min(c["sinks"], pos + 1 - c["window"])


def work(c):
    if c["op"] == "verify":
        # one row of the target's probabilities a sequence, and the draft's where one is
        # rejected (about three sequences in four here); two products a token
        rows = c["seqs"] * (1.75 if c["draft_probs"] else 1.0)
        return {"bytes": rows * c["vocab"] * 4, "flops": rows * c["vocab"] * 2}
    item = 4 if c["type"] == "f32" else 2
    n, length = new_tokens(c), lengths(c)
    row, tokens = c["kv_heads"] * c["head_dim"], sum(n)
    if c["op"] == "append":
        q = tokens * c["heads"] * c["head_dim"]
        span = sum(a - b for a, b in zip(length, _first_pages(c)))
        moved = 2 * q * item + 2 * tokens * row * (item + 1) + tokens * c["head_dim"] * 4  # rotated, written, tables
        return {"bytes": moved + 2 * span * row * (1 + item), "flops": 3 * q + 6 * tokens * row}
    pairs = sum(_visible(c, a - k + i) for a, k in zip(length, n) for i in (range(k) if k < 64 else ()))
    pairs += sum(k * (_visible(c, a - k) + _visible(c, a - 1)) // 2 for a, k in zip(length, n) if k >= 64)
    keys = sum(min(a, _visible(c, a - k) + k - 1) for a, k in zip(length, n) if k)
    return {"bytes": 2 * keys * row + 8 * (keys // c["page"]) * c["kv_heads"] + 2 * tokens * c["heads"] * c["head_dim"] * item,
            "flops": 4 * pairs * c["heads"] * c["head_dim"]}


# ---- inputs ------------------------------------------------------------------------


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _pages(g, n_pages, c):
    """Pages of quantized normal values whose size differs from page to page."""
    x = _normal(g, n_pages, c["kv_heads"], c["page"], c["head_dim"])
    x *= torch.exp(0.25 * _normal(g, n_pages, c["kv_heads"], 1, 1))
    scale = x.abs().amax((2, 3)) / 127
    codes = torch.round(x / scale[:, :, None, None]).add_(128).to(torch.uint8)
    return codes, scale


def _rotation(c, positions):
    half = c["head_dim"] // 2
    freq = 500000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "verify":
        B, K, V = c["seqs"], c["drafts"], c["vocab"]
        logits = _normal(g, B, K + 1, V, scale=3.0)
        s = {"case": c, "target": torch.softmax(logits, -1)}
        if c["draft_probs"]:  # a draft model that is mostly of the target's opinion
            s["draft"] = torch.softmax(logits[:, :K] + _normal(g, B, K, V, scale=0.7), -1)
            s["tokens"] = torch.multinomial(s["draft"].reshape(B * K, V), 1, generator=g).reshape(B, K).int()
        else:  # tokens looked up in the context, no probabilities: mostly the likeliest
            s["draft"] = None
            s["tokens"] = logits[:, :K].argmax(-1).int()
        s["drafted"] = _ints([K - (b % 2 if K > 1 else 0) for b in range(B)])
        s["uniform"] = torch.rand(B, K + 1, generator=g, device=DEV)
        return s
    kind = torch.float32 if c["type"] == "f32" else torch.bfloat16
    n, length = new_tokens(c), lengths(c)
    tokens, starts = sum(n), [sum(n[:i]) for i in range(c["seqs"] + 1)]
    per_seq = [-(-a // c["page"]) for a in length]
    n_pages = sum(per_seq) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table, at = [], 0
    for p in per_seq:
        table.append(order[at:at + p] + [-1] * (max(per_seq) - p))
        at += p
    s = {"case": c, "q_start": _ints(starts), "kv_len": _ints(length), "page_table": _ints(table), "n_tokens": tokens}
    s["k_codes"], s["k_scale"] = _pages(g, n_pages, c)
    s["v_codes"], s["v_scale"] = _pages(g, n_pages, c)
    s["q"] = _normal(g, tokens, c["heads"] * c["head_dim"], scale=1.5).to(kind)
    if c["op"] == "append":
        s["k"] = _normal(g, tokens, c["kv_heads"] * c["head_dim"]).to(kind)
        s["v"] = _normal(g, tokens, c["kv_heads"] * c["head_dim"]).to(kind)
        s["cos"], s["sin"] = _rotation(c, c["longest"])
        s["first"] = _ints(_first_pages(c))
        s["count"] = max(a - b for a, b in zip(length, _first_pages(c)))
    if own:  # the handles a server keeps: the cache, and the step's batch with its workspace
        if "squirrel-rs_b200" not in sys.path:
            sys.path.insert(0, "squirrel-rs_b200")
        from sqb200 import paged
        s["cache"] = paged.PagedCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        s["batch"] = paged.PagedBatch(s["q_start"], s["kv_len"], s["page_table"], n_tokens=tokens, max_new=max(n))
    return s


# ---- one pass ----------------------------------------------------------------------


def run(s):
    c = s["case"]
    if own:
        if "squirrel-rs_b200" not in sys.path:
            sys.path.insert(0, "squirrel-rs_b200")
        from sqb200 import paged, speculative
        if c["op"] == "verify":
            accepted, tokens = speculative.verify_drafts(s["target"], s["draft"], s["tokens"], s["uniform"], s["drafted"])
            return {"accepted": accepted, "tokens": tokens}
        if c["op"] == "append":
            q = paged.append(s["cache"], s["batch"], s["k"], s["v"], s["cos"], s["sin"], q=s["q"])
            k, v = paged.read(s["cache"], s["batch"], s["first"], s["count"], dtype=s["k"].dtype)
            return {"q": q, "k": k, "v": v}
        return {"out": paged.attention(s["cache"], s["batch"], s["q"], window=c["window"], sinks=c["sinks"])}
    return {"append": plain_append, "attention": plain_attention, "verify": plain_verify}[c["op"]](s)


def _token_places(s):
    """Sequence and position of every new token."""
    q_start, kv_len = s["q_start"].long(), s["kv_len"].long()
    t = torch.arange(s["n_tokens"], device=DEV)
    b = torch.searchsorted(q_start, t, right=True) - 1
    return b, kv_len[b] - q_start[b + 1] + t


def _rotated(x, cos, sin, pos, head_dim):
    """Interleaved pairs (2j, 2j+1) rotated by the angles of the row's position."""
    x = x.float().view(x.shape[0], -1, head_dim // 2, 2)
    a, b, c, s = x[..., 0], x[..., 1], cos[pos][:, None], sin[pos][:, None]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(2)


def _store(codes, scale, x, pages, slot, touched, kept):
    """Quantize rows x [tokens, kv_heads, head_dim] into (pages, slot). `touched` are the
    pages that get new tokens, `kept` whether such a page holds earlier ones: its scale
    only grows, and its earlier codes follow it."""
    limit = torch.full((), 127.0, device=DEV)
    need = torch.zeros_like(scale).scatter_reduce_(0, pages[:, None].expand(-1, scale.shape[1]), x.abs().amax(2) / limit, "amax")
    old = scale[touched] * kept[:, None]
    now = torch.maximum(old, need[touched])
    inverse = torch.where(now > 0, 1 / now, 0.0)
    ratio = (old * inverse)[:, :, None, None]
    codes[touched] = (torch.round((codes[touched].float() - 128) * ratio) + 128).to(torch.uint8)
    scale[touched] = now
    grid = torch.round(x * torch.where(scale > 0, 1 / scale, 0.0)[pages][:, :, None])
    codes[pages, :, slot] = (grid.clamp(-127, 127) + 128).to(torch.uint8)


def plain_append(s):
    c = s["case"]
    hd, page = c["head_dim"], c["page"]
    b, pos = _token_places(s)
    q = _rotated(s["q"], s["cos"], s["sin"], pos, hd).flatten(1).to(s["q"].dtype)
    k = _rotated(s["k"], s["cos"], s["sin"], pos, hd)
    v = s["v"].float().view(-1, c["kv_heads"], hd)
    table = s["page_table"].long()
    pages = table[b, pos // page]
    # each sequence's pages from its first new token on; the others stand on its first one
    start, end = s["kv_len"].long() - s["q_start"].long().diff(), s["kv_len"].long()
    at = start[:, None] // page + torch.arange((s["count"] + page - 1) // page, device=DEV)
    live = (at * page < end[:, None]) & (start < end)[:, None]
    touched = table.gather(1, at.clamp(max=table.shape[1] - 1))[live]
    kept = (at * page < start[:, None])[live]
    for codes, scale, x in ((s["k_codes"], s["k_scale"], k), (s["v_codes"], s["v_scale"], v)):
        _store(codes, scale, x, pages, pos % page, touched, kept)
    at = s["first"].long()[:, None] + torch.arange(s["count"], device=DEV)
    live = at < end[:, None]
    where = table.gather(1, (at // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    out = []
    for codes, scale in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])):
        x = (codes[where, :, at % page].float() - 128) * scale[where][..., None] * live[..., None, None]
        out.append(x.flatten(2).to(s["k"].dtype))
    return {"q": q, "k": out[0], "v": out[1]}


def plain_attention(s):
    c = s["case"]
    hd, page, group = c["head_dim"], c["page"], c["heads"] // c["kv_heads"]
    b, pos = _token_places(s)
    row = torch.arange(s["n_tokens"], device=DEV) - s["q_start"].long()[b]
    most = max(new_tokens(c))
    q = torch.zeros(c["seqs"], most, c["kv_heads"], group, hd, device=DEV)
    q[b, row] = s["q"].float().view(-1, c["kv_heads"], group, hd)
    where = torch.full((c["seqs"], most), -1, device=DEV)
    where[b, row] = pos
    table = s["page_table"].long().clamp(min=0)

    def dense(codes, scale):  # [seqs, kv_heads, positions, head_dim]
        x = (codes[table].float() - 128) * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(c["seqs"], c["kv_heads"], -1, hd)

    key = torch.arange(table.shape[1] * page, device=DEV)
    seen = key <= where[..., None]
    if c["window"]:
        seen &= (key > where[..., None] - c["window"]) | (key < c["sinks"])
    q = q.permute(0, 2, 3, 1, 4).reshape(c["seqs"], c["kv_heads"], group * most, hd) / math.sqrt(hd)
    score = (q @ dense(s["k_codes"], s["k_scale"]).transpose(2, 3)).view(c["seqs"], c["kv_heads"], group, most, -1)
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    weight = (weight / torch.where(total > 0, total, 1.0)).view(c["seqs"], c["kv_heads"], group * most, -1)
    out = (weight @ dense(s["v_codes"], s["v_scale"])).view(c["seqs"], c["kv_heads"], group, most, hd)
    return {"out": out.permute(0, 3, 1, 2, 4)[b, row].flatten(1).to(s["q"].dtype)}


def _weights(x):
    """Probabilities as whole numbers, so that their sums do not depend on an order."""
    return (torch.where(x > 0, x.clamp(max=1.0), 0.0) * 2.0**FRACTION_BITS).to(torch.int64)


def plain_verify(s):
    target, draft, tokens, n, u = s["target"], s["draft"], s["tokens"].long(), s["drafted"].long(), s["uniform"]
    B, K = tokens.shape
    p = target[:, :K].gather(2, tokens[..., None])[..., 0]
    q = draft.gather(2, tokens[..., None])[..., 0] if draft is not None else torch.ones_like(p)
    place = torch.arange(K, device=DEV)
    accepted = ((u[:, :K] * q < p) & (place < n[:, None])).long().cumprod(1).sum(1)
    rejected, rows = accepted < n, torch.arange(B, device=DEV)
    at = accepted.clamp(max=K - 1)
    full = target[rows, accepted]
    if draft is not None:
        left = full - draft[rows, at]
    else:  # the draft was certain of its token
        left = full.scatter(1, tokens[rows, at][:, None], 0.0)
    weight = _weights(torch.where(rejected[:, None], left, full))
    weight = torch.where((weight.sum(1) > 0)[:, None], weight, _weights(full))
    total = weight.sum(1)
    step = 2**UNIFORM_BITS
    part = (u[:, K].clamp(min=0) * step).to(torch.int64).clamp(max=step - 1)
    goal = part * (total // step) + part * (total % step) // step
    token = (weight.cumsum(1) <= goal[:, None]).sum(1)
    token = torch.where(total > 0, token, -1)
    place = torch.arange(K + 1, device=DEV)
    padded = torch.cat((tokens, torch.zeros_like(tokens[:, :1])), 1)
    out = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], token[:, None], -1))
    return {"accepted": accepted.int(), "tokens": out.int()}


# ---- the definitions in 64 bits ----------------------------------------------------


def exact(case, seed):
    if case["op"] == "verify":  # whole numbers alone: the plain form is exact
        return None
    s = prepare(case, seed)
    return exact_append(s) if case["op"] == "append" else exact_attention(s)


def exact_append(s):
    """Sequence by sequence and page by page."""
    c = s["case"]
    hd, page, kvh = c["head_dim"], c["page"], c["kv_heads"]
    angle = torch.complex(s["cos"].double(), s["sin"].double())
    starts, length, table, first = (s[n].tolist() for n in ("q_start", "kv_len", "page_table", "first"))
    q_out, read = [], {n: torch.zeros(c["seqs"], s["count"], kvh, hd, dtype=torch.float64, device=DEV) for n in "kv"}
    for b in range(c["seqs"]):
        a, e = starts[b], starts[b + 1]
        p0 = length[b] - (e - a)
        turn = angle[p0:length[b], None]

        def spin(x, heads):
            z = torch.view_as_complex(x[a:e].double().reshape(e - a, heads, hd // 2, 2).contiguous())
            return torch.view_as_real(z * turn).reshape(e - a, heads, hd)

        q_out.append(spin(s["q"], c["heads"]).flatten(1))
        for name, x in (("k", spin(s["k"], kvh)), ("v", s["v"][a:e].double().view(e - a, kvh, hd))):
            codes, scale = s[name + "_codes"], s[name + "_scale"]
            for p in range(first[b], length[b], page):
                here = table[b][p // page]
                end = min(p + page, length[b])
                held = max(p0 - p, 0)
                rows = x[max(p, p0) - p0:end - p0].transpose(0, 1)  # [kv_heads, new rows, head_dim]
                before = (codes[here, :, :held].double() - 128)
                was = scale[here].double() if held else torch.zeros(kvh, dtype=torch.float64, device=DEV)
                now = torch.maximum(was, rows.abs().amax((1, 2)) / 127) if rows.shape[1] else was
                step = now[:, None, None]
                block = torch.cat((torch.round(before * was[:, None, None] / step), torch.round(rows / step)), 1) * step
                read[name][b, p - first[b]:end - first[b]] = torch.nan_to_num(block).transpose(0, 1)
    return {"q": torch.cat(q_out), "k": read["k"].flatten(2), "v": read["v"].flatten(2)}


def exact_attention(s):
    """Sequence by sequence, one key/value head and a few queries at a time."""
    c = s["case"]
    hd, group = c["head_dim"], c["heads"] // c["kv_heads"]
    starts, length, table = (s[n].tolist() for n in ("q_start", "kv_len", "page_table"))
    out = torch.zeros(s["n_tokens"], c["heads"], hd, dtype=torch.float64, device=DEV)
    for b in range(c["seqs"]):
        a, e, end = starts[b], starts[b + 1], length[b]
        if a == e:
            continue
        pages = torch.tensor(table[b][:-(-end // c["page"])], device=DEV)
        for h in range(c["kv_heads"]):
            k, v = (((s[n + "_codes"][pages, h].double() - 128) * s[n + "_scale"][pages, h].double()[:, None, None])
                    .reshape(-1, hd)[:end] for n in "kv")
            for i in range(a, e, 512):
                j = min(i + 512, e)
                pos = torch.arange(end - (e - i), end - (e - j), device=DEV)[:, None]
                key = torch.arange(end, device=DEV)
                hidden = key > pos
                if c["window"]:
                    hidden |= (key <= pos - c["window"]) & (key >= c["sinks"])
                q = s["q"][i:j].double().view(j - i, c["heads"], hd)[:, h * group:(h + 1) * group]
                score = torch.einsum("igd,kd->igk", q, k) / math.sqrt(hd)
                score = score.masked_fill(hidden[:, None], float("-inf"))
                out[i:j, h * group:(h + 1) * group] = torch.einsum("igk,kd->igd", torch.softmax(score, -1), v)
    return {"out": out.flatten(1)}
