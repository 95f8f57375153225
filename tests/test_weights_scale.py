"""CPU test: both forms of the attention weights refuse the scales that the prompt
attention and its wrappers refuse, before any launch."""
import ctypes

import pytest

from gpu_offloading_amd import _lib
from test_operator_plans import _weights


@pytest.mark.parametrize("scale", [0.0, -0.125, float("inf"), float("nan")])
def test_scales_that_are_not_positive_and_finite(scale):
    lib = _lib.load()
    _, s, *_ = _weights(lib, [5], [40], 4, 2, 128)
    sc = ctypes.c_float(scale)
    assert lib.kvc_batch_attention_weights_run(
        ctypes.byref(s), 64, None, 0, 64, 512, 64, 64, 4096, 256, 4, 64, 3, 1, sc, 64, None, None,
        0, None, None) == 1
    # (a batch of nothing: refused for its scale alone)
    assert lib.kvc_decode_attention_weights(
        64, 512, 64, 64, 4096, 256, 4, 64, 64, 3, 64, 0, 4, 2, 128, 16, 1, sc, 64, None, None, 0,
        None, None) == 1
    assert b"sm_scale" in lib.kvc_last_error()
