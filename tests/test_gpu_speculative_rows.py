"""Verification over slices of wider probability tensors, on the GPU."""
import numpy as np
import pytest

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
