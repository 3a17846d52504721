"""Softmax scales that the attention entry refuses because their product with log2 e is no FP32 number (no GPU)."""
import ctypes

import pytest

P, L, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float


@pytest.mark.parametrize("scale", [2.3e38, 2.4e38, 2.9e38])
def test_scales_whose_base_2_form_overflows_are_refused(ops, scale):
    one = P(16)
    code = ops.libci8.ci8_kv4_attention(one, L(1024), one, one, one, one, one, one, 4, 2, 3, 9, 16, 8, 2, 128, F(scale), P(0))
    assert code == 1
