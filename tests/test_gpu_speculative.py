"""Verification of drafted tokens on the GPU: whole numbers, equal to the restated rule
(paged_oracle.verify), and the distribution of what comes out."""
import numpy as np
import pytest

import paged_oracle as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def case(seed, n, k, vocab, spread=3.0):
    rng = np.random.default_rng(seed)
    logits = rng.standard_normal((n, k + 1, vocab)) * spread
    target = softmax(logits)
    draft = softmax(logits[:, :k] + rng.standard_normal((n, k, vocab)) * 0.7)
    tokens = np.array([[rng.choice(vocab, p=draft[b, i].astype(np.float64) / draft[b, i].sum(dtype=np.float64))
                        for i in range(k)] for b in range(n)], np.int32).reshape(n, k)
    return rng, target, draft, tokens, rng.random((n, k + 1), np.float32)


def check(target, draft, tokens, uniform, n_draft=None):
    from sqb200 import speculative
    n, k = tokens.shape
    acc, out = speculative.verify_drafts(dev(target), dev(draft) if draft is not None else None, dev(tokens),
                                         dev(uniform), dev(n_draft) if n_draft is not None else None)
    want_acc, want = P.verify(target, draft, tokens, n_draft if n_draft is not None else [k] * n, uniform)
    np.testing.assert_array_equal(acc.cpu().numpy(), want_acc)
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    return want_acc, want


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("n,k,vocab", [(1, 1, 1), (1, 4, 7), (5, 3, 1000), (3, 40, 333), (9, 2, 4099), (2, 5, 128256),
                                       (4, 0, 513)])
def test_verify(gpu_lib, n, k, vocab, with_draft):
    rng, target, draft, tokens, uniform = case(vocab + k, n, k, vocab)
    n_draft = rng.integers(0, k + 1, n).astype(np.int32)
    check(target, draft if with_draft else None, tokens, uniform, n_draft)
    check(target, draft if with_draft else None, tokens, uniform)


def test_verify_greedy_rows(gpu_lib):
    """One-hot targets: drafts are accepted exactly while they equal the target's choice."""
    rng = np.random.default_rng(3)
    want = rng.integers(0, 50, (6, 4))
    target = np.eye(50, dtype=np.float32)[want]
    tokens = want[:, :3].astype(np.int32).copy()
    tokens[1, 0] += 1
    tokens[2, 2] -= 1
    tokens %= 50
    acc, out = check(target, None, tokens, rng.random((6, 4), np.float32))
    assert acc.tolist() == [3, 0, 2, 3, 3, 3]
    assert out[0].tolist() == want[0].tolist() and out[1, 0] == want[1, 0]


def test_verify_edges(gpu_lib):
    """Uniforms of 0, nearly 1 and beyond; a remainder without mass; rows without mass, with
    NaN, with negative and large values; tokens outside the vocabulary; equal rows."""
    n, k, v = 9, 2, 40
    rng, target, draft, tokens, uniform = case(8, n, k, v)
    uniform[0], uniform[1], uniform[2] = 0, np.float32(1) - np.float32(2**-24), 1.5
    target[3, 0], draft[3, 0], uniform[3, 0] = 0, 0, 0.5       # rejected, nothing left, no target either
    target[4, 0] = draft[4, 0]
    draft[4, 0, tokens[4, 0]] *= 4                             # rejected with little mass left
    uniform[4, 0] = 0.9
    target[5, 1, 3:9], target[5, 2, 0] = np.nan, np.nan
    target[6, 2] = -1
    target[6, 2, 11] = 0.25                                    # the only mass
    target[7] *= 1000
    target[8], draft[8] = target[8, 0], target[8, 0]           # equal: everything is accepted
    with np.errstate(invalid="ignore"):
        check(target, draft, tokens, uniform)
    bad = tokens.copy()
    bad[0, 0], bad[1, 1] = v, -1
    from sqb200 import speculative
    acc, _ = speculative.verify_drafts(dev(target), dev(draft), dev(bad), dev(uniform))
    assert acc[0] == 0 and acc[1] <= 1  # such a token is rejected


def test_verify_remainder_without_mass_falls_back(gpu_lib):
    """target <= draft everywhere (the target's row sums to less): drawn from the target."""
    target = np.full((1, 2, 64), 1 / 128, np.float32)
    draft = np.full((1, 1, 64), 1 / 64, np.float32)
    acc, out = check(target, draft, np.int32([[5]]), np.float32([[0.75, 0.5]]))
    assert acc[0] == 0 and out[0, 0] == 32


def test_verify_strided_rows(gpu_lib):
    """Rows padded to a wider stride that is no multiple of four elements."""
    from sqb200 import speculative
    _, target, draft, tokens, uniform = case(5, 3, 2, 1001)
    want = speculative.verify_drafts(dev(target), dev(draft), dev(tokens), dev(uniform))
    for pad in (1, 3, 7):
        t = torch.full((3, 3, 1001 + pad), 9.0, device="cuda")
        d = torch.full((3, 2, 1001 + pad), 0.0, device="cuda")
        t[..., :1001], d[..., :1001] = dev(target), dev(draft)
        got = speculative.verify_drafts(t[..., :1001], d[..., :1001], dev(tokens), dev(uniform))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_verify_keeps_the_targets_distribution(gpu_lib):
    """Drafted from q and verified, first tokens are distributed as the target: over N draws a
    frequency is within 5 standard deviations sqrt(p (1 - p) / N) of its probability."""
    from sqb200 import speculative
    n, v = 40000, 12
    rng = np.random.default_rng(17)
    p, q = softmax(rng.standard_normal(v) * 1.5), softmax(rng.standard_normal(v) * 1.5)
    target = np.broadcast_to(p, (n, 2, v)).copy()
    draft = np.broadcast_to(q, (n, 1, v)).copy()
    tokens = rng.choice(v, (n, 1), p=q.astype(np.float64) / q.sum(dtype=np.float64)).astype(np.int32)
    _, out = speculative.verify_drafts(dev(target), dev(draft), dev(tokens), dev(rng.random((n, 2), np.float32)))
    freq = np.bincount(out[:, 0].cpu().numpy(), minlength=v) / n
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-9).all()
