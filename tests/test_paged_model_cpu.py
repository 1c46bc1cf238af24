"""The parts of sqb200.paged_model that need no GPU: the GGUF reader against the writer, the
rotation table against the oracle's frequencies."""
import numpy as np
import pytest

from sqb200 import gguf_synth as G

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("wtype", ["q8_0", "q4_0", "bf16"])
def test_reader_finds_what_was_written(wtype):
    from sqb200 import paged_model as M
    path = G.ensure_gguf("tiny", wtype)
    meta, tensors = M.read_gguf(path)
    spec = G.SPECS["tiny"]
    assert meta["llama.block_count"] == spec["layers"] and meta["llama.attention.head_count_kv"] == spec["kv_heads"]
    want = G.tensor_list(spec, G.TYPE_NAMES[wtype])
    assert [(n, d, t) for n, (d, t, _) in tensors.items()] == [(n, d, t) for n, d, t in want]
    for i, (name, dims, kind) in enumerate(want):
        data = tensors[name][2]
        assert data.size == G.tensor_nbytes(int(np.prod(dims)), kind)
        if kind == G.F32:
            assert (data.view(np.float32) == 1).all()
        else:
            rng = np.random.Generator(np.random.PCG64(np.random.SeedSequence([0, i])))
            x = rng.standard_normal(dims[0], dtype=np.float32) * np.float32(0.02)
            assert np.array_equal(data[:G.tensor_nbytes(dims[0], kind)], G.quantize(x, kind))


def test_reader_refuses_other_files(tmp_path):
    from sqb200 import paged_model as M
    p = tmp_path / "x.gguf"
    p.write_bytes(b"GGML" + bytes(100))
    with pytest.raises(ValueError):
        M.read_gguf(str(p))
    p.write_bytes(b"GGUF" + (2).to_bytes(4, "little") + bytes(100))
    with pytest.raises(ValueError):
        M.read_gguf(str(p))


def test_rotation_table_scales_like_llama3():
    """Short wavelengths keep their frequency, long ones are divided by the factor, those between
    lie between (models/llama/config.rs:83-127)."""
    from sqb200 import lib
    from sqb200 import paged_model as M
    c = lib.LlamaConfig(head_dim=64, rope_base=500000.0, rope_factor=32.0, rope_low_freq=1.0, rope_high_freq=4.0,
                        rope_orig_ctx=8192.0)
    cos, sin = M.rope_table(c, 3, "cpu")
    assert cos.shape == (3, 32) and (cos[0] == 1).all() and (sin[0] == 0).all()
    plain = 500000.0 ** (-np.arange(32) / 32)
    freq = np.arctan2(sin[1].double().numpy(), cos[1].double().numpy())
    wave = 2 * np.pi / plain
    short, long = wave < 8192 / 4, wave > 8192
    assert np.allclose(freq[short], plain[short], rtol=1e-5) and np.allclose(freq[long], plain[long] / 32, rtol=1e-3)
    between = ~short & ~long
    assert between.any() and (freq[between] <= plain[between]).all() and (freq[between] >= plain[between] / 32).all()
