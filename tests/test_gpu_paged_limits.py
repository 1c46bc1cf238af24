"""The paged attention at the edges of what its arguments and batches may say, against tests/paged_oracle.py."""
import numpy as np
import pytest

import paged_oracle as P
from test_gpu_paged import KINDS, Setup, dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_short_prompts_leave_the_second_row_tile_idle(gpu_lib, hd, kind):
    """Row tiles of up to 128 rows and one or two key blocks, some of more rows between them: a thread block goes
    through several of them while one of its product warps has nothing to do. The result, and equal bits on every call."""
    from sqb200 import paged
    news = [20 + i % 12 if i % 7 else 33 + i for i in range(300)]
    s = Setup(21, 8, hd, 32, news, [n + (i * 11) % 60 for i, n in enumerate(news)])
    q = s.rows(32 * hd, kind, 1.5)
    first = paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind]))
    for _ in range(100):
        assert torch.equal(paged.attention(s.dcache, s.batch, dev(q).to(KINDS[kind])), first)
    s.check_attention(32, kind, q=q)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("sinks", [0, 3])
@pytest.mark.parametrize("window", [255, 256, 257, 2**30, 2**31 - 16, 2**31 - 1, 2**31 + 5, 2**40])
def test_windows_as_long_as_the_table_and_longer(gpu_lib, window, sinks, kind):
    """A window that holds every position there can be hides nothing, whatever its size. (The table here has 16
    pages of 16: the oracle takes the window as it is.)"""
    for heads, news, lens in ((8, [1, 3], [1, 9]), (8, [40, 90, 1, 2], [40, 100, 240, 2])):
        Setup(22, 2, 64, 16, news, lens).check_attention(heads, kind, window=window, sinks=sinks)
