"""The paged attention at the edges of what its arguments and batches may say, against tests/paged_oracle.py."""
import pytest

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
