"""A Llama over the paged 8-bit cache: several sequences at once, with tokens drafted by the
model's own first blocks. It runs the operators of a batched server together as they are
meant: append and attention in every block (sqb200.paged), verification after the last
(sqb200.speculative); everything else is the op level (sqb200.lib).

    python squirrel-rs_b200/sqb200/paged_model.py --spec small --seqs 4 --tokens 32 --draft 4

The reference serves one sequence with an f32 cache (models/llama/model.rs:45-97,
text_generator.rs:38-101); the block's arithmetic here is the same (models/llama/layers.rs:
24-109), the cache's 8 bits apart.
"""
import argparse
import os
import struct
import sys

import numpy as np
import torch

if __package__ in (None, ""):  # run as a file
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from sqb200 import lib, paged, speculative  # noqa: E402


def read_gguf(path):
    """(metadata: U32, F32 and strings; tensors: name -> (dims, type, bytes as a numpy view))
    of a GGUF v3 file (file_parser/gguf_file.rs:22-49)."""
    data = np.memmap(path, np.uint8, "r")
    at = 0

    def take(fmt):
        nonlocal at
        v = struct.unpack_from("<" + fmt, data, at)[0]
        at += struct.calcsize("<" + fmt)
        return v

    def text():
        nonlocal at
        n = take("Q")
        s = bytes(data[at:at + n]).decode()
        at += n
        return s

    if bytes(data[:4]) != b"GGUF":
        raise ValueError(f"{path}: not a GGUF file")
    at = 4
    if take("I") != 3:
        raise ValueError(f"{path}: GGUF version 3 is wanted")
    n_tensors, n_meta = take("Q"), take("Q")
    meta = {}
    for _ in range(n_meta):
        key, kind = text(), take("I")
        if kind not in (4, 6, 8):
            raise ValueError(f"{path}: metadata {key} of type {kind}")
        meta[key] = text() if kind == 8 else take("I" if kind == 4 else "f")
    infos = []
    for _ in range(n_tensors):
        name = text()
        dims = [take("Q") for _ in range(take("I"))]
        infos.append((name, dims, take("I"), take("Q")))
    base = -(-at // 32) * 32
    sizes = {lib.F32: lambda n: 4 * n, **{t: (lambda n, b=b: n // 32 * b) for t, b in lib.BLOCK_BYTES.items()}}
    return meta, {name: (dims, kind, data[base + off:base + off + sizes[kind](int(np.prod(dims)))])
                  for name, dims, kind, off in infos}


def rope_table(config, positions, device):
    """cos, sin [positions, head_dim / 2] of the llama3-scaled frequencies
    (models/llama/config.rs:83-127, kernels/rope.rs:7-36), in float32 like the reference."""
    f = np.float32
    j = np.arange(config.head_dim // 2, dtype=f)
    freq = np.power(f(config.rope_base), f(-2) * j * (f(1) / f(config.head_dim))).astype(f)
    wave = f(6.28318548202514648438) / freq
    smooth = (f(config.rope_orig_ctx) / wave - f(config.rope_low_freq)) / f(config.rope_high_freq - config.rope_low_freq)
    slow = freq / f(config.rope_factor)
    mixed = (f(1) - smooth) * slow + smooth * freq
    freq = np.where(wave > config.rope_orig_ctx / config.rope_low_freq, slow,
                    np.where(wave >= config.rope_orig_ctx / config.rope_high_freq, mixed, freq)).astype(f)
    angle = np.arange(positions, dtype=f)[:, None] * freq
    return torch.from_numpy(np.cos(angle)).to(device), torch.from_numpy(np.sin(angle)).to(device)


class Sequence:
    """Tokens of one sequence; the first `held` of them are in the cache, in `pages`."""

    def __init__(self, tokens):
        self.tokens = [int(t) for t in tokens]
        self.held, self.pages = 0, []


class PagedLlama:
    def __init__(self, path, n_pages, page=64, device="cuda"):
        """The GGUF file's weights in their native blocks on the GPU, and a pool of n_pages
        pages in every block's cache, shared by all sequences."""
        meta, tensors = read_gguf(path)
        c = self.config = lib.LlamaConfig()
        for field, key in (("n_blocks", "block_count"), ("embed_dim", "embedding_length"), ("ffn_dim", "feed_forward_length"),
                           ("n_heads", "attention.head_count"), ("n_kv_heads", "attention.head_count_kv"),
                           ("head_dim", "rope.dimension_count"), ("vocab_size", "vocab_size"),
                           ("context_length", "context_length"), ("rope_base", "rope.freq_base"),
                           ("rms_eps", "attention.layer_norm_rms_epsilon")):
            setattr(c, field, meta["llama." + key])
        for field, key, default in (("rope_factor", "factor", 32.0), ("rope_low_freq", "low_freq_factor", 1.0),
                                    ("rope_high_freq", "high_freq_factor", 4.0),
                                    ("rope_orig_ctx", "original_context_length", 8192)):
            setattr(c, field, meta.get("llama.rope.scaling." + key, default))

        def weight(name):
            dims, kind, data = tensors[name]
            t = torch.from_numpy(np.array(data)).to(device)
            return (t.view(torch.float32) if kind == lib.F32 else t), kind

        self.embd, self.embd_type = weight("token_embd.weight")
        self.head, self.head_type = weight("output.weight") if "output.weight" in tensors else (self.embd, self.embd_type)
        self.out_norm = weight("output_norm.weight")[0]
        names = ("attn_norm", "attn_q", "attn_k", "attn_v", "attn_output", "ffn_norm", "ffn_gate", "ffn_up", "ffn_down")
        self.blocks = [{n: weight(f"blk.{i}.{n}.weight")[0] for n in names} for i in range(c.n_blocks)]
        c.weight_type = tensors["blk.0.attn_q.weight"][1]
        self.caches = [paged.PagedCache.empty(n_pages, c.n_kv_heads, c.head_dim, page, device) for _ in range(c.n_blocks)]
        self.page, self.device = page, device
        self.free = list(range(n_pages))[::-1]
        self.cos, self.sin = rope_table(c, min(c.context_length, n_pages * page), device)

    def _step(self, seqs, news):
        """The batch of the next news[i] tokens of each sequence, with pages for them."""
        if max(s.held + n for s, n in zip(seqs, news)) > self.cos.shape[0]:
            raise lib.KernelError(19, f"a sequence would pass the rotation table's {self.cos.shape[0]} positions")
        for s, n in zip(seqs, news):
            while len(s.pages) * self.page < s.held + n:
                if not self.free:
                    raise lib.KernelError(19, "no free page in the cache")
                s.pages.append(self.free.pop())
        width = max(1, max(len(s.pages) for s in seqs))
        table = np.full((len(seqs), width), -1, np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(s.pages)] = s.pages

        def dev(v):
            return torch.tensor(v, dtype=torch.int32, device=self.device)

        starts = np.concatenate([[0], np.cumsum(news)])
        return paged.PagedBatch(dev(starts), dev([s.held + n for s, n in zip(seqs, news)]), dev(table), int(starts[-1]),
                                max(news))

    def hidden(self, ids, batch, n_blocks):
        """The rows' hidden states after the first n_blocks blocks (models/llama/layers.rs:81-109)."""
        c, kind = self.config, self.config.weight_type
        q, kv = c.n_heads * c.head_dim, c.n_kv_heads * c.head_dim
        x = lib.embed(ids, self.embd, self.embd_type, c.embed_dim, c.vocab_size)
        for w, cache in zip(self.blocks[:n_blocks], self.caches):
            h = lib.rms_norm(x, w["attn_norm"], c.rms_eps)
            xq, xk, xv = lib.linear_shared(h, [w["attn_q"], w["attn_k"], w["attn_v"]], kind, [q, kv, kv])
            paged.append(cache, batch, xk, xv, self.cos, self.sin, q=xq, q_out=xq)
            x = lib.elementwise_add(x, lib.linear(paged.attention(cache, batch, xq), w["attn_output"], kind, c.embed_dim))
            h = lib.rms_norm(x, w["ffn_norm"], c.rms_eps)
            gate, up = lib.linear_shared(h, [w["ffn_gate"], w["ffn_up"]], kind, [c.ffn_dim, c.ffn_dim])
            x = lib.elementwise_add(x, lib.linear(lib.silu_mul(gate, up), w["ffn_down"], kind, c.embed_dim))
        return x

    def logits(self, x):
        c = self.config
        return lib.linear(lib.rms_norm(x.contiguous(), self.out_norm, c.rms_eps), self.head, self.head_type, c.vocab_size)

    def forward(self, seqs, news, n_blocks=None):
        """Logits [sum(news), vocab] of the next news[i] tokens of each sequence (they must be
        known), which the cache then holds as positions held .. held + news[i] - 1; the
        caller says with Sequence.held how many of them stay."""
        ids = [t for s, n in zip(seqs, news) for t in s.tokens[s.held:s.held + n]]
        ids = torch.tensor(ids, dtype=torch.int32, device=self.device)
        return self.logits(self.hidden(ids, self._step(seqs, news), n_blocks or self.config.n_blocks))

    def release(self, seq):
        self.free += seq.pages
        seq.pages, seq.held = [], 0


def probabilities(logits, temperature):
    """softmax(logits / temperature); temperature 0: all on the first largest."""
    if temperature == 0:
        return torch.nn.functional.one_hot(logits.argmax(-1), logits.shape[-1]).float()
    return torch.softmax(logits / temperature, -1)


def spread(rows, counts):
    """[n, max(counts), vocab] from rows [sum(counts), vocab] of n sequences, zeros behind the shorter ones."""
    n, most, vocab = len(counts), max(counts), rows.shape[1]
    if min(counts) == most:
        return rows.view(n, most, vocab)
    out = rows.new_zeros((n * most, vocab))
    out[[b * most + i for b, c in enumerate(counts) for i in range(c)]] = rows
    return out.view(n, most, vocab)


def generate(model, prompts, max_tokens, draft=4, draft_blocks=1, temperature=1.0, generator=None):
    """max_tokens new tokens of each prompt: in every round the first draft_blocks blocks
    draft `draft` tokens one after the other (fewer where a sequence wants fewer), the whole
    model scores them in one pass, and the accepted ones and one more are kept. A sequence
    leaves the rounds with its last token, and never holds more than len(prompt) + max_tokens - 1
    positions. With draft=0 a plain batched decode. Returns (token lists, share of
    drafted tokens accepted); raises CacheFull without pages or positions for them, and what
    the kernels recorded (paged.status, lib.wait_status)."""
    seqs = [Sequence(p) for p in prompts]
    if not all(s.tokens for s in seqs):
        raise lib.KernelError(3, "a prompt without tokens")
    vocab = model.config.vocab_size
    uniform = lambda n, k: torch.rand(n, k, device=model.device, generator=generator)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=model.device)  # noqa: E731
    try:
        # the prompts but their last tokens, which every round starts with
        news = [len(s.tokens) - 1 for s in seqs]
        if max(news, default=0):
            model.forward(seqs, news)
            for s, k in zip(seqs, news):
                s.held += k
        want = [len(s.tokens) + max_tokens for s in seqs]
        drafted = taken = 0
        while True:
            live = [(s, w - len(s.tokens)) for s, w in zip(seqs, want) if len(s.tokens) < w]
            if not live:
                break
            left = [k for _, k in live]
            live = [s for s, _ in live]
            n, most = len(live), [min(draft, k - 1) for k in left]  # one token is drawn after the drafts
            probs = []
            for i in range(max(most)):
                on = [s for s, k in zip(live, most) if k > i]
                p = probabilities(model.forward(on, [i + 1] * len(on), draft_blocks).view(len(on), i + 1, vocab)[:, -1],
                                  temperature)
                _, token = speculative.verify_drafts(p[:, None], None, ints([[]] * len(on)), uniform(len(on), 1))  # drawn from p
                for s, t in zip(on, token[:, 0].tolist()):
                    s.tokens.append(t)
                probs.append(p.new_zeros((n, vocab)).index_copy_(0, ints([b for b, k in enumerate(most) if k > i]).long(), p)
                             if len(on) < n else p)
            target = probabilities(model.forward(live, [k + 1 for k in most]), temperature)
            tokens = ints([s.tokens[s.held + 1:] + [0] * (max(most) - k) for s, k in zip(live, most)])
            accepted, out = speculative.verify_drafts(spread(target, [k + 1 for k in most]),
                                                      torch.stack(probs, 1) if probs else None, tokens,
                                                      uniform(n, max(most) + 1), ints(most))
            for s, k, m, row in zip(live, accepted.tolist(), most, out.tolist()):
                s.tokens[s.held + 1:] = row[:k + 1]  # the accepted drafts and the drawn token
                s.held += k + 1
                drafted, taken = drafted + m, taken + k
        # the last round's results are on the host: every kernel of the call has run
        paged.status()
        lib.wait_status()
    finally:
        for s in seqs:
            model.release(s)
    return [s.tokens for s in seqs], taken / max(drafted, 1)


def main():
    from sqb200 import gguf_synth as g
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--spec", default="small", choices=list(g.SPECS))
    ap.add_argument("--type", default="q8_0", choices=list(g.TYPE_NAMES))
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=40)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--draft", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=1.0)
    a = ap.parse_args()
    model = PagedLlama(g.ensure_gguf(a.spec, a.type), n_pages=a.seqs * (-(-(a.prompt + a.tokens + a.draft + 1) // 64) + 1))
    prompts = [g.prompt_ids(a.prompt + i, seed=i, high=g.SPECS[a.spec]["vocab"]) for i in range(a.seqs)]
    rng = torch.Generator("cuda").manual_seed(0)
    out, share = generate(model, prompts, a.tokens, a.draft, temperature=a.temperature, generator=rng)
    torch.cuda.synchronize()
    paged.status()
    for p, t in zip(prompts, out):
        print(*t[len(p):])
    print(f"{share:.0%} of the drafted tokens accepted")


if __name__ == "__main__":
    main()
