"""Sizes that the attention entry refuses because a token's place in a sequence would not fit its arithmetic (no GPU)."""
import ctypes

import pytest

P, L, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float


@pytest.mark.parametrize("page", [16, 64, 256])
def test_tables_of_more_than_2_to_the_30_tokens_are_refused(ops, page):
    one, width = P(16), 2 ** 30 // page + 1
    code = ops.libci8.ci8_kv4_attention(one, L(1024), one, one, one, one, one, one, 4, 2, width, 9, page, 8, 2, 128, F(0.1), P(0))
    assert code == 1
