"""What verify_drafts makes of its tensors' strides, on the host: _probs looks at shape and strides
first, so host tensors show which rows it takes (they pass all but the last check) and which not."""
import pytest

torch = pytest.importorskip("torch")


def layout(x):
    return f"{tuple(x.shape)}by{x.stride()}" if torch.is_tensor(x) else str(x)


def outcome(t, n, rows, vocab):
    """"taken", or the kind and message of the refusal."""
    from sqb200 import speculative
    from sqb200.lib import KernelError
    with pytest.raises(KernelError) as e:
        speculative._probs(t, n, rows, vocab, 0, "draft")
    return "taken" if "CUDA tensor" in str(e.value) else (e.value.kind, str(e.value))


@pytest.mark.parametrize("t,n,rows", [
    (torch.zeros(1000).expand(4, 5, 1000), 4, 5),           # one distribution for all places
    (torch.zeros(1, 1, 1000).expand(1, 4, 1000), 1, 4),
    (torch.zeros(1, 1, 1000).expand(3, 1, 1000), 3, 1),
    (torch.zeros(3, 1, 1000).expand(3, 2, 1000), 3, 2),     # one for each sequence's places
    (torch.zeros(1, 2, 1000).expand(3, 2, 1000), 3, 2),     # one for each place of all sequences
    (torch.zeros(2000).as_strided((1, 3, 1000), (0, 500, 1)), 1, 3),
    (torch.zeros(2000).as_strided((2, 1, 1000), (999, 1, 1)), 2, 1),
], ids=layout)
def test_rows_that_lie_over_one_another_are_refused(t, n, rows):
    kind, message = outcome(t, n, rows, 1000)
    assert kind == "ShapeMismatch" and "one stride between rows" in message


def test_other_layouts_are_refused():
    x = torch.zeros(3, 4, 20)
    assert outcome(x.transpose(1, 2), 3, 20, 4)[0] == "ShapeMismatch"     # a row's elements apart
    assert outcome(x[..., ::2], 3, 4, 10)[0] == "ShapeMismatch"
    assert outcome(x[:, :2], 3, 2, 20)[0] == "ShapeMismatch"              # two strides between rows
    assert outcome(x, 3, 5, 20)[0] == "ShapeMismatch"
    assert outcome(x.double(), 3, 4, 20)[0] == "InvalidType"


@pytest.mark.parametrize("t,n,rows,vocab", [
    (torch.zeros(3, 4, 20), 3, 4, 20),
    (torch.zeros(3, 4, 23)[..., :20], 3, 4, 20),
    (torch.zeros(3, 4, 20)[:, -1:], 3, 1, 20),              # the last place of each sequence
    (torch.zeros(1, 4, 20)[:, 1:3], 1, 2, 20),
    (torch.zeros(1, 4, 20)[:, 2:3], 1, 1, 20),
    (torch.zeros(3, 0, 20), 3, 0, 20),
    (torch.zeros(3, 4, 1).expand(3, 4, 1), 3, 4, 1),
], ids=layout)
def test_rows_one_stride_apart_are_taken(t, n, rows, vocab):
    assert outcome(t, n, rows, vocab) == "taken"
