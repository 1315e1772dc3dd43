"""The QK-norm operator loads its tables 16 bytes at a time: others are refused, without a GPU."""
import ctypes

import pytest


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("which", ["cos", "sin"])
def test_tables_that_are_not_16_byte_aligned_are_refused(lib, n, which):
    from modern_llm_v1_b200 import _lib

    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 255) & ~255
    cos, sin = (p + 4, p) if which == "cos" else (p, p + 8)
    B, T, H, D, big = 1, 4, 2, 64, 1 << 30
    if n == 1:
        assert lib.b200attn_rope_norm_fwd(p, 0, 1, p, 0, p, p, cos, sin, B, T, H, D, 1e-5, None) == _lib.ERR_ALIGNMENT
        assert lib.b200attn_rope_norm_bwd(p, 0, p, 0, 1, p, p, cos, sin, p, p, B, T, H, D, p, big, None) == _lib.ERR_ALIGNMENT
    else:
        assert lib.b200attn_rope_norm_fwd_qk(p, p, 0, 1, p, p, 0, p, p, p, p, cos, sin, B, T, H, 1, D, 1e-5, None) == _lib.ERR_ALIGNMENT
        assert lib.b200attn_rope_norm_bwd_qk(p, p, 0, p, p, 0, 1, p, p, p, p, cos, sin, p, p, p, p, B, T, H, 1, D, p, big, None) == _lib.ERR_ALIGNMENT
