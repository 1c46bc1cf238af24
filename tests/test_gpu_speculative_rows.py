"""Verification over slices of wider probability tensors, on the GPU."""
import numpy as np
import pytest

import paged_oracle as P
from test_gpu_speculative import case, dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("vocab", [40, 1001])
def test_verify_slices_of_the_places(gpu_lib, vocab):
    """The last place of each sequence, and some places of one sequence: the ids of the contiguous copies."""
    from sqb200 import speculative
    _, target, _, _, uniform = case(5, 6, 3, vocab)
    wide = dev(target)
    none = torch.zeros((6, 0), dtype=torch.int32, device="cuda")
    u = dev(uniform[:, :1])
    got = speculative.verify_drafts(wide[:, -1:], None, none, u)
    want = speculative.verify_drafts(wide[:, -1:].contiguous(), None, none, u)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    tokens = dev(np.int32([[1]]))
    got = speculative.verify_drafts(wide[2:3, 1:3], None, tokens, dev(uniform[2:3, :2]))
    want = speculative.verify_drafts(wide[2:3, 1:3].contiguous(), None, tokens, dev(uniform[2:3, :2]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("vocab", [1, 3, 130])
def test_verify_small_vocabularies(gpu_lib, vocab):
    """Rows that leave most blocks of a cluster nothing to read: their sums are exchanged as soon as they start. Many
    clusters, many more than run at once, on every call the same ids."""
    from sqb200 import speculative
    rng = np.random.default_rng(vocab)
    n, k = 3000, 2
    target, draft = (rng.random((n, r, vocab), np.float32) / vocab for r in (k + 1, k))
    tokens, uniform = rng.integers(0, vocab, (n, k)).astype(np.int32), rng.random((n, k + 1), np.float32)
    acc, out = P.verify(target, draft, tokens, [k] * n, uniform)
    args = [dev(x) for x in (target, draft, tokens, uniform)]
    for _ in range(5):
        got_acc, got = speculative.verify_drafts(*args)
        np.testing.assert_array_equal(got_acc.cpu().numpy(), acc)
        np.testing.assert_array_equal(got.cpu().numpy(), out)


@pytest.mark.parametrize("k", [0, 3])
def test_verify_no_sequences(gpu_lib, k):
    from sqb200 import speculative
    z = lambda *s, **kw: torch.zeros(s, device="cuda", **kw)  # noqa: E731
    for draft in (None, z(0, k, 50)):
        acc, out = speculative.verify_drafts(z(0, k + 1, 50), draft, z(0, k, dtype=torch.int32), z(0, k + 1),
                                             z(0, dtype=torch.int32))
        assert acc.shape == (0,) and out.shape == (0, k + 1)
