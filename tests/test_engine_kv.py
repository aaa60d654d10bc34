"""Engines that are opened with a choice of KV cache."""
import ctypes
import dataclasses

import numpy as np
import pytest

from leap_b200 import LeapError, ModelConfig, Transformer, _native
from leap_b200.modelfile import write_v1

CFG = ModelConfig(dim=512, hidden_dim=1024, n_layers=2, n_heads=8, n_kv_heads=4, vocab_size=500, seq_len=128)


def test_an_unknown_kind_is_refused_before_the_model_is_touched():
    with pytest.raises(ValueError, match="kv must be"):
        Transformer.create("/nonexistent/model.bin", kv="q9")
    with pytest.raises(ValueError, match="kv must be"):
        Transformer.synthetic(CFG, False, kv="q9")
    with pytest.raises(LeapError, match="open file"):
        Transformer.create("/nonexistent/model.bin", kv="q8")
    lib = _native.lib()
    h = ctypes.c_void_p()
    c = _native.ModelConfigC(*CFG.as_tuple(), 0, 0, 1)
    for kind in (-1, 2):
        assert lib.leap_engine_open_kv(b"/nonexistent/model.bin", 0, 0, -1, 0.0, 0, kind,
                                       ctypes.byref(h)) == _native.LEAP_ERR_INVALID
        assert b"kv kind" in lib.leap_last_error() and not h.value
        assert lib.leap_engine_synthetic_kv(ctypes.byref(c), 0, 0, 0, -1, 0.0, 0, kind,
                                            ctypes.byref(h)) == _native.LEAP_ERR_INVALID
        assert b"kv kind" in lib.leap_last_error() and not h.value
    assert lib.leap_engine_open_kv(None, 0, 0, -1, 0.0, 0, 1, ctypes.byref(h)) == _native.LEAP_ERR_INVALID
    assert lib.leap_engine_synthetic_kv(None, 0, 0, 0, -1, 0.0, 0, 1, ctypes.byref(h)) == _native.LEAP_ERR_INVALID


@pytest.mark.gpu
def test_opened_and_replaced_are_the_same(cuda, tmp_path):
    path = str(tmp_path / "m.bin")
    write_v1(path, CFG, seed=1)
    toks = np.random.default_rng(0).integers(0, 500, 40)
    got = []
    for kv, then in (("q8", None), ("f32", "q8"), ("f32", None), ("q8", "f32")):
        with Transformer.create(path, kv=kv) as t:
            if then:
                t.set_kv(then)
            t.prefill(toks[:-1])
            got.append((t.forward(int(toks[-1]), 39), t.device_bytes()))
    for a, b in ((0, 1), (2, 3)):
        np.testing.assert_array_equal(got[a][0], got[b][0])
        assert got[a][1] == got[b][1]
    assert got[0][1] != got[2][1]


@pytest.mark.gpu
def test_a_context_that_only_8_bit_rows_fit(cuda):
    """FP32 rows of this length are more than the GPU's memory."""
    import torch
    free, total = torch.cuda.mem_get_info()
    cfg = ModelConfig(dim=1024, hidden_dim=256, n_layers=64, n_heads=8, n_kv_heads=8, vocab_size=256, seq_len=64)
    row = 2 * cfg.n_layers * cfg.n_kv_heads * 128
    cfg = dataclasses.replace(cfg, seq_len=int(1.1 * total / (4 * row)))
    if free < 0.45 * total:
        pytest.skip("less than half of the memory is free")
    with Transformer.synthetic(cfg, True, kv="q8") as t:
        assert t.device_bytes() < 0.4 * total
        out = t.forward(3, 0)
        assert np.isfinite(out).all()


@pytest.mark.gpu
def test_replacing_the_cache_reports_what_went_wrong_before(cuda):
    """A token id outside the vocabulary, found on the device: the error is not
    lost with the cache's context, and the engine keeps what it had."""
    import torch
    with Transformer.synthetic(CFG, False, seed=2) as t:
        t.bind_torch_stream()
        before = t.device_bytes()
        want = t.forward(7, 0)
        x = torch.empty(1, CFG.dim, device="cuda")
        t.embed_device(torch.tensor([CFG.vocab_size], dtype=torch.int32, device="cuda"), x)
        with pytest.raises(LeapError, match="token id"):
            t.set_kv("q8")
        assert t.device_bytes() == before
        np.testing.assert_array_equal(t.forward(7, 0), want)
        t.set_kv("q8")
        assert t.device_bytes() != before


@pytest.mark.gpu
@pytest.mark.parametrize("first,then", [("f32", "q8"), ("q8", "f32"), ("f32", "f32")])
def test_device_bytes_after_a_replaced_cache(cuda, first, then):
    """What prefill allocated beside the old cache is gone with it."""
    with Transformer.synthetic(CFG, False, kv=then) as t:
        want = t.device_bytes()
    with Transformer.synthetic(CFG, False, kv=first) as t:
        t.prefill(np.arange(100))
        t.set_kv(then)
        assert t.device_bytes() == want
