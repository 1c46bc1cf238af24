"""The paged Llama (sqb200.paged_model): its logits against the model with the f32 cache, and
generation with drafted tokens against generation without."""
import numpy as np
import pytest

from sqb200 import gguf_synth as G

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def load(spec="small", wtype="q8_0", n_pages=24, page=64):
    from sqb200 import paged_model as M
    return M.PagedLlama(G.ensure_gguf(spec, wtype), n_pages, page)


@pytest.mark.parametrize("spec,wtype,page", [("small", "q8_0", 64), ("small", "bf16", 16), ("tiny", "q4_0", 16)])
def test_logits_follow_the_f32_cache(gpu_lib, spec, wtype, page):
    """A prompt in ragged pieces beside other sequences: every piece's last logits within the
    8-bit cache's noise of the f32 cache's. A value is off by up to amax / 254 of its page,
    under 2% of a unit normal value; averaged over many values a block adds under 1% of the
    residual stream's size, and logits of these models have a size of about 0.5: 0.03 in all."""
    from sqb200 import lib, paged
    from sqb200 import paged_model as M
    vocab = G.SPECS[spec]["vocab"]
    model = load(spec, wtype, page=page)
    ref = lib.Model(G.ensure_gguf(spec, wtype))
    prompts = [G.prompt_ids(n, seed=n, high=vocab) for n in (90, 3, 41)]
    seqs = [M.Sequence(p) for p in prompts]
    ctxs = [ref.new_context(128) for _ in prompts]
    for news in ([70, 1, 0], [1, 0, 40], [19, 2, 1]):
        logits = model.forward(seqs, news)
        at = 0
        for s, c, n in zip(seqs, ctxs, news):
            if n:
                c.forward(np.uint32(s.tokens[s.held:s.held + n]))
                got = logits[at + n - 1].cpu().numpy()
                assert np.abs(got - c.logits()).max() <= 0.03
            s.held += n
            at += n
    torch.cuda.synchronize()
    paged.status()
    for c in ctxs:
        c.close()
    ref.close()


def test_drafting_everything_accepts_everything(gpu_lib):
    """With all blocks drafting, draft and target are the same model up to the order of sums:
    nearly every draft is accepted. At temperature 0 every id is the f32-cache model's choice
    after what precedes it, or within twice the logits' noise (0.03 above) of it."""
    from sqb200 import lib
    from sqb200 import paged_model as M
    prompts = [G.prompt_ids(n, seed=n, high=4096) for n in (20, 1, 33)]
    blocks = G.SPECS["small"]["layers"]
    ref = lib.Model(G.ensure_gguf("small", "q8_0"))
    for draft in (0, 3):
        ids, share = M.generate(load(), prompts, 24, draft=draft, draft_blocks=blocks, temperature=0)
        assert share > 0.9 or not draft
        for p, t in zip(prompts, ids):
            ctx = ref.new_context(128)
            ctx.forward(p)
            for token in t[len(p):]:
                logits = ctx.logits()
                assert logits[token] >= logits.max() - 0.06
                ctx.forward(np.uint32([token]))
            ctx.close()
    ref.close()
    _, share = M.generate(load(), prompts, 24, draft=3, draft_blocks=blocks, temperature=1.0)
    assert share > 0.9


def test_generation_with_drafts_is_reproducible_and_returns_its_pages(gpu_lib):
    from sqb200 import paged_model as M
    model = load()
    prompts = [G.prompt_ids(n, seed=n, high=4096) for n in (30, 64, 7, 1)]
    outs = []
    for _ in range(2):
        rng = torch.Generator("cuda").manual_seed(5)
        outs.append(M.generate(model, prompts, 20, draft=4, draft_blocks=1, temperature=1.0, generator=rng))
        assert sorted(model.free) == list(range(24))
    assert outs[0] == outs[1]
    assert all(len(t) == len(p) + 20 and t[:len(p)] == [int(x) for x in p] for t, p in zip(outs[0][0], prompts))


def test_a_full_pool_is_an_error(gpu_lib):
    from sqb200 import lib
    from sqb200 import paged_model as M
    model = load(n_pages=2)
    with pytest.raises(lib.KernelError) as e:
        model.forward([M.Sequence(G.prompt_ids(200, high=4096))], [200])
    assert e.value.kind == "CacheFull"
