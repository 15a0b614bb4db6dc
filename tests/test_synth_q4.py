"""The Q4_0 quantizer of b2q.synth against gguf-py's."""
import numpy as np
import pytest

from b2q import synth


def test_q4_0_matches_gguf():
    gguf = pytest.importorskip("gguf")
    typ = gguf.GGMLQuantizationType.Q4_0
    rng = np.random.default_rng(0)
    w = rng.standard_normal((40, 128)).astype(np.float32)
    w[3] = 0
    w[4, :32] = 1.0
    w[5, 7] = -100.0
    q = synth.quantize_q4_0(w)
    np.testing.assert_array_equal(q, gguf.quants.quantize(w, typ))
    np.testing.assert_array_equal(synth.dequantize_q4_0(q, 128), gguf.quants.dequantize(q, typ))


def test_q4_0_error_is_half_a_step():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((16, 64)).astype(np.float32)
    back = synth.dequantize_q4_0(synth.quantize_q4_0(w), 64)
    step = np.abs(w.reshape(-1, 32)).max(1, keepdims=True) / 8
    # the largest value's opposite is cut at +7 steps: a whole step; the scale is rounded to 11 bits
    assert (np.abs(back - w).reshape(-1, 32) <= step * (1 + 2.0 ** -7)).all()


def test_columns_must_be_whole_blocks():
    with pytest.raises(ValueError):
        synth.quantize_q4_0(np.zeros((2, 33), np.float32))
