"""Plain forms of the paged 8-bit cache's operators for the tests: append restated step by
step in numpy f32 (every operation rounded on its own, so codes and scales must be equal),
attention and the token draw from their definitions in 64 bits and whole numbers."""
import math

import numpy as np


def rotation(positions, head_dim):
    freq = 500000.0 ** (-np.arange(head_dim // 2) / (head_dim // 2))
    a = np.arange(positions)[:, None] * freq
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotate(x, cos, sin):
    """x [rows, heads, head_dim] f32, cos / sin [rows, head_dim / 2]: interleaved pairs."""
    a, b, c, s = x[..., 0::2], x[..., 1::2], cos[:, None], sin[:, None]
    out = np.empty_like(x)
    out[..., 0::2] = a * c - b * s
    out[..., 1::2] = a * s + b * c
    return out


def store(codes, scale, rows, offset):
    """Write rows [n, head_dim] f32 into one page and head from `offset` on: codes [page,
    head_dim] uint8 in place; returns the new scale."""
    f = np.float32
    held = offset > 0
    was = f(scale) if held else f(0)
    size = np.abs(rows)
    size = size[np.isfinite(size)]
    need = (size.max() if size.size else f(0)) / f(127)
    now = max(was, f(need))
    with np.errstate(over="ignore", invalid="ignore"):
        inv = min(f(1) / now, np.finfo(f).max) if now > 0 else f(0)
        if held and now > was:
            ratio = was * inv
            codes[:offset] = np.clip(np.rint((codes[:offset].astype(f) - f(128)) * ratio), -127, 127) + 128
        y = np.rint(rows * inv)
        y = np.clip(np.where(np.isnan(y), f(0), y), -127, 127)
    codes[offset:offset + len(rows)] = (y + 128).astype(np.uint8)
    return now


def append(cache, q_start, kv_len, table, k, v, cos, sin):
    """cache: dict of numpy arrays k, v, ks, vs, changed in place."""
    page, hd = cache["k"].shape[2:]
    heads = cache["k"].shape[1]
    for b in range(len(kv_len)):
        a, e = q_start[b], q_start[b + 1]
        p0 = kv_len[b] - (e - a)
        if a == e:
            continue
        kr = rotate(k[a:e].reshape(e - a, heads, hd), cos[p0:kv_len[b]], sin[p0:kv_len[b]])
        vr = v[a:e].reshape(e - a, heads, hd)
        for p in range(p0 // page, (kv_len[b] - 1) // page + 1):
            lo, hi = max(p * page, p0), min((p + 1) * page, kv_len[b])
            at = table[b][p]
            for g in range(heads):
                for codes, scales, x in (("k", "ks", kr), ("v", "vs", vr)):
                    cache[scales][at, g] = store(cache[codes][at, g], cache[scales][at, g], x[lo - p0:hi - p0, g],
                                                 lo - p * page)


def values(codes, scales, pages, head, n):
    """[n, head_dim] f64 of one sequence and kv head."""
    x = (codes[pages, head].astype(np.float64) - 128) * scales[pages, head].astype(np.float64)[:, None, None]
    return x.reshape(-1, codes.shape[3])[:n]


def attention(cache, q_start, kv_len, table, q, heads, window=0, sinks=0, scale=None):
    """(out, spread): the f64 result [rows, heads, head_dim] and, for the bounds, per row and
    head the largest sum |q_d k_d| * scale over the seen keys and the largest |v| seen."""
    kvh, page, hd = cache["k"].shape[1:]
    group = heads // kvh
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = np.zeros((q.shape[0], heads, hd))
    size = np.zeros((q.shape[0], heads, 2))
    for b in range(len(kv_len)):
        a, e, n = q_start[b], q_start[b + 1], kv_len[b]
        if a == e or n == 0:
            continue
        pages = np.asarray(table[b][:-(-n // page)])
        pos = np.arange(n - (e - a), n)[:, None]
        key = np.arange(n)[None]
        seen = key <= pos
        if window:
            seen &= (key > pos - window) | (key < sinks)
        for g in range(kvh):
            k = values(cache["k"], cache["ks"], pages, g, n)
            v = values(cache["v"], cache["vs"], pages, g, n)
            for h in range(g * group, (g + 1) * group):
                x = q[a:e].reshape(e - a, heads, hd)[:, h].astype(np.float64)
                s = np.where(seen, x @ k.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                w = np.exp(s - np.where(np.isfinite(top), top, 0))
                total = w.sum(1, keepdims=True)
                w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
                out[a:e, h] = w @ v
                size[a:e, h, 0] = np.where(seen, np.abs(x) @ np.abs(k).T * abs(scale), 0).max(1)
                size[a:e, h, 1] = np.where(seen, np.abs(v).max(1)[None], 0).max(1)
    return out, size


def bound(out, size, dtype):
    """How far an output may be off. A score is q.k with q as two f16 terms (22 bits) or
    one (bf16 rows: exact) and products summed in f32: |ds| <= 2^-20 sum |q_d k_d| scale.
    That moves the weights' shares by at most 2 ds in all, so the output by 2 ds max |v|.
    The weights themselves are 22-bit (f32 rows: 2^-20 with the sums) or f16 (2^-11)
    numbers. A bf16 output is rounded once: 2^-8 |out|."""
    ds, top = size[..., 0:1] * 2.0**-20, size[..., 1:2]
    if dtype == "f32":
        return top * (2 * ds + 2.0**-19) + 1e-30
    return top * (2 * ds + 2.0**-10) + 2.0**-8 * np.abs(out) + 1e-30


def verify(target, draft, tokens, n_draft, uniform):
    n, k = tokens.shape
    accepted, out = np.zeros(n, np.int64), np.full((n, k + 1), -1, np.int64)
    for b in range(n):
        i = 0
        while i < n_draft[b]:
            x = tokens[b, i]
            q = draft[b, i, x] if draft is not None else np.float32(1)
            if not uniform[b, i] * q < target[b, i, x]:
                break
            i += 1
        out[b, :i], accepted[b] = tokens[b, :i], i
        full = target[b, i]
        left = full.copy()
        if i < n_draft[b]:
            if draft is not None:
                left = full - draft[b, i]
            else:
                left[tokens[b, i]] = 0

        def weights(x):
            return [int(min(float(p), 1.0) * 2**38) if p > 0 else 0 for p in x]

        w = weights(left)
        if sum(w) == 0:
            w = weights(full)
        total = sum(w)
        if total:
            part = min(max(int(float(uniform[b, k]) * 2**24), 0), 2**24 - 1)
            goal, run = part * total >> 24, 0
            for j, x in enumerate(w):
                run += x
                if run > goal:
                    out[b, i] = j
                    break
    return accepted, out
