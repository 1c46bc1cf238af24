"""The bindings of the paged cache and the verification, on the host."""
import ctypes as C
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

NAMES = ["sq_paged_append", "sq_paged_attention", "sq_paged_read", "sq_verify_drafts", "sq_paged_status"]


@pytest.mark.parametrize("name", NAMES)
def test_calls_give_up_the_interpreter_lock(name):
    """They can wait for the GPU; other threads go on meanwhile."""
    from sqb200 import paged
    assert not paged._fn(name)._flags_ & C._FUNCFLAG_PYTHONAPI


class Elsewhere:
    """A tensor's face, on GPU 1."""

    def __init__(self, *shape, dtype=torch.float32):
        self.t = torch.zeros(shape, dtype=dtype)
        self.shape, self.dtype, self.stride, self.is_contiguous = self.t.shape, dtype, self.t.stride, self.t.is_contiguous
        self.dim, self.numel, self.new_empty, self.is_cuda = self.t.dim, self.t.numel, self.t.new_empty, True

    def get_device(self):
        return 1

    def data_ptr(self):
        return 256


def refused(call, *args, **kw):
    from sqb200.lib import KernelError
    with pytest.raises(KernelError) as e:
        call(*args, **kw)
    return e.value.kind, str(e.value)


def test_tensors_of_another_device_are_refused(monkeypatch):
    """The kernels run on the current device: what lies elsewhere must not be handed to them."""
    from sqb200 import paged, speculative
    monkeypatch.setattr(paged, "_device", lambda: 0)
    monkeypatch.setattr(speculative, "_device", lambda: 0)
    monkeypatch.setattr(paged, "_fn", lambda name: pytest.fail(name))
    monkeypatch.setattr(speculative, "_fn", lambda name: lambda *a: pytest.fail(name))
    monkeypatch.setattr(speculative, "_raw_stream", lambda d: 0)

    def world(cache, batch):
        return (SimpleNamespace(device=cache, row=128, half=32, head_dim=64), SimpleNamespace(device=batch, n_tokens=3, n_seqs=2))

    k, table = Elsewhere(3, 128), Elsewhere(9, 32)
    for c, b in ((1, 0), (0, 1), (1, 1)):
        assert "current CUDA device" in refused(paged.append, *world(c, b), k, k, table, table)[1]
        assert "current CUDA device" in refused(paged.attention, *world(c, b), k)[1]
        assert "current CUDA device" in refused(paged.read, *world(c, b), Elsewhere(2, dtype=torch.int32), 4)[1]
    assert refused(paged.append, *world(0, 0), k, k, table, table) == (
        "InvalidArgument", "InvalidArgument: k: a CUDA tensor of the current device is wanted")
    assert refused(paged.attention, *world(0, 0), k)[0] == "InvalidArgument"
    assert refused(paged.read, *world(0, 0), Elsewhere(2, dtype=torch.int32), 4)[0] == "ShapeMismatch"
    args = [Elsewhere(2, 4, 50), None, Elsewhere(2, 3, dtype=torch.int32), Elsewhere(2, 4)]
    assert refused(speculative.verify_drafts, *args)[0] == "InvalidArgument"


@pytest.mark.parametrize("count", [-1, 2**31])
def test_read_refuses_counts_out_of_range(monkeypatch, count):
    from sqb200 import paged
    monkeypatch.setattr(paged, "_device", lambda: 1)
    first = Elsewhere(2, dtype=torch.int32)
    world = SimpleNamespace(device=1, row=128, half=32, head_dim=64, like={torch.float32: torch.zeros(0)}), SimpleNamespace(
        device=1, n_tokens=3, n_seqs=2)
    assert refused(paged.read, *world, first, count)[0] == "ShapeMismatch"
