"""What sqb200.paged_model.generate asks of its model, on the host: a model that goes by a rule in place of
the GPU's, the restated verification (paged_oracle.verify) in place of the kernel, the pool's real pages."""
from types import SimpleNamespace

import numpy as np
import pytest

import paged_oracle as P

torch = pytest.importorskip("torch")

VOCAB = 8


@pytest.fixture
def world(monkeypatch):
    from sqb200 import lib, paged, paged_model, speculative

    def verify(target, draft, tokens, uniform, n_draft=None):
        n, k = tokens.shape
        acc, out = P.verify(target.numpy(), draft.numpy() if draft is not None else None, tokens.numpy(),
                            n_draft.tolist() if n_draft is not None else [k] * n, uniform.numpy())
        return torch.from_numpy(acc).int(), torch.from_numpy(out).int()

    calls = []
    monkeypatch.setattr(speculative, "verify_drafts", verify)
    monkeypatch.setattr(paged, "PagedBatch", lambda *a: a)
    monkeypatch.setattr(paged, "status", lambda clear=True: calls.append("status"))
    monkeypatch.setattr(lib, "wait_status", lambda clear=True: calls.append("wait_status"))

    class Model(paged_model.PagedLlama):
        """The next token is the same again; drafting says so of even tokens alone."""

        def __init__(self, n_pages, page=4, positions=1000):
            self.page, self.device, self.free = page, "cpu", list(range(n_pages))
            self.cos = torch.zeros(positions, 1)
            self.config = SimpleNamespace(vocab_size=VOCAB, n_blocks=3)
            self.most, self.rows = {}, []

        def forward(self, seqs, news, n_blocks=None):
            self._step(seqs, news)
            self.rows.append(sum(news))
            ids = []
            for s, n in zip(seqs, news):
                self.most[id(s)] = max(self.most.get(id(s), 0), s.held + n)
                assert len(s.tokens) >= s.held + n
                ids += [t + 2 * (n_blocks is not None and t % 2) for t in s.tokens[s.held:s.held + n]]
            return torch.from_numpy(np.eye(VOCAB, dtype=np.float32)[np.array(ids, int) % VOCAB])

    return SimpleNamespace(Model=Model, generate=paged_model.generate, calls=calls)


@pytest.mark.parametrize("draft", [0, 1, 4, 9])
@pytest.mark.parametrize("max_tokens", [1, 2, 17])
def test_sequences_that_are_done_leave_the_rounds(world, draft, max_tokens):
    """One sequence takes every draft, one none: the first is done long before. The pool has the pages of
    the wanted tokens and no more."""
    prompts = [[2] * 3, [1] * 6, [4], [3] * 9]
    pages = sum(-(-(len(p) + max_tokens - 1) // 4) for p in prompts)
    model = world.Model(pages)
    out, share = world.generate(model, prompts, max_tokens, draft=draft, temperature=0)
    assert out == [p + p[:1] * max_tokens for p in prompts]
    assert sorted(model.most.values()) == sorted(len(p) + max_tokens - 1 for p in prompts)
    assert len(model.free) == pages
    if draft and max_tokens > 1:
        # the even sequences draft what they want but one a round, all accepted; the odd ones nothing accepted
        even = odd = 0
        left = max_tokens
        while left:
            even += min(draft, left - 1)
            left -= min(draft, left - 1) + 1
        odd = sum(min(draft, left - 1) for left in range(1, max_tokens + 1))
        assert share == pytest.approx(even / (even + odd))


@pytest.mark.parametrize("call", [0, 1, 3])
def test_pages_come_back_from_a_call_that_fails(world, call):
    """Whatever raises: no page, a drafting pass, a scoring pass."""
    from sqb200.lib import KernelError

    class Failing(world.Model):
        def forward(self, *a):
            out = super().forward(*a)
            if len(self.rows) > call:
                raise RuntimeError("as told")
            return out

    model = Failing(20)
    with pytest.raises(RuntimeError):
        world.generate(model, [[2] * 7, [3] * 9], 5, draft=2, temperature=0)
    assert sorted(model.free) == list(range(20))
    model = world.Model(3)
    with pytest.raises(KernelError) as e:
        world.generate(model, [[2] * 7, [3] * 9], 5, draft=2, temperature=0)
    assert e.value.kind == "CacheFull" and sorted(model.free) == list(range(3))


def test_positions_past_the_rotation_table_are_an_error(world):
    """Their keys would be left out of the cache. As many positions as there are is taken."""
    from sqb200.lib import KernelError
    out, _ = world.generate(world.Model(20, positions=11), [[2] * 7], 5, draft=3, temperature=0)
    assert out == [[2] * 12]
    model = world.Model(20, positions=10)
    with pytest.raises(KernelError) as e:
        world.generate(model, [[2] * 7], 5, draft=3, temperature=0)
    assert e.value.kind == "CacheFull" and "10 positions" in str(e.value) and len(model.free) == 20


def test_what_the_kernels_recorded_is_asked_for(world, monkeypatch):
    from sqb200 import paged
    world.generate(world.Model(20), [[2] * 7], 5, temperature=0)
    assert world.calls == ["status", "wait_status"]

    def raises(clear=True):
        raise RuntimeError("recorded")

    monkeypatch.setattr(paged, "status", raises)
    with pytest.raises(RuntimeError, match="recorded"):
        world.generate(world.Model(20), [[2] * 7], 5, temperature=0)


def test_empty_prompts_are_refused_and_no_prompts_are_none(world):
    from sqb200.lib import KernelError
    model = world.Model(20)
    with pytest.raises(KernelError) as e:
        world.generate(model, [[2, 2], []], 5, temperature=0)
    assert e.value.kind == "EmptyInput" and len(model.free) == 20 and not model.rows
    assert world.generate(model, [], 5, temperature=0) == ([], 0)
