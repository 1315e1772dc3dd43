"""What the rotary calls refuse, without a GPU."""
import ctypes

import pytest
import torch


def _buf():
    buf = ctypes.create_string_buffer(8192)
    return buf, (ctypes.addressof(buf) + 255) & ~255


def test_c_abi_refuses_before_any_cuda_call(lib):
    from modern_llm_v1_b200 import _lib

    keep, p = _buf()
    f = lambda R=64, pairs=1, D=64, n_pos=8, T=4, pos=None, gq=None, gk=None, rq=None, x=p, cos=p: lib.b200attn_rotary_fwd(  # noqa: E731
        x, p, 0, 1, p, p, 0, rq, rq, gq, gk, cos, p, pos, n_pos, R, pairs, 1, T, 2, 1, D, 1e-5, None)
    assert f(D=32, R=32) == _lib.ERR_UNSUPPORTED
    for R in (0, -16, 8, 24, 80):
        assert f(R=R) == _lib.ERR_INVALID_ARG
    assert f(pairs=2) == _lib.ERR_INVALID_ARG
    assert f(n_pos=3) == _lib.ERR_INVALID_ARG  # fewer rows than tokens
    assert f(n_pos=0, pos=p) == _lib.ERR_INVALID_ARG
    assert f(gq=p, gk=None, rq=p) == _lib.ERR_INVALID_ARG
    assert f(gq=p, gk=p) == _lib.ERR_INVALID_ARG  # no rstd
    assert f(x=None) == _lib.ERR_INVALID_ARG
    assert f(x=p + 2) == _lib.ERR_ALIGNMENT
    assert f(cos=p + 4) == _lib.ERR_ALIGNMENT
    b = lambda gamma, x, ws, n: lib.b200attn_rotary_bwd(p, p, 0, x, x, 0, 1, gamma, gamma, gamma, gamma, p, p, None, 8, 64, 1, p, p, gamma,  # noqa: E731
                                                        gamma, 1, 4, 2, 1, 64, ws, n, None)
    assert b(p, None, p, 1 << 30) == _lib.ERR_INVALID_ARG
    assert b(p, p, None, 0) == _lib.ERR_WORKSPACE
    assert b(p, p, p, 16) == _lib.ERR_WORKSPACE
    t = lib.b200attn_rotary_table
    assert t(0, 64, 1e4, 0, 1.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 63, 1e4, 0, 1.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 64, 0.0, 0, 1.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 64, 1e4, 4, 1.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 64, 1e4, 1, 0.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 2, 1e4, 2, 2.0, 0.0, 0.0, 0.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 64, 1e4, 3, 2.0, 0.0, 32.0, 1.0, p, p, None) == _lib.ERR_INVALID_ARG
    assert t(8, 64, 1e4, 3, 2.0, 99.0, 1.0, 1.0, p, p, None) == _lib.ERR_INVALID_ARG
    a = lambda pos0=0, row0=0, n_new=1, n_pos=8, L_cap=4, gk=p, R=64: lib.b200attn_kv_append_rotary(  # noqa: E731
        p, p, p, 0, p, p, p, None, p, gk, p, p, n_pos, R, 0, None, pos0, None, row0, 1, n_new, L_cap, 2, 1, 64, 1e-5, None)
    assert a(pos0=8) == a(pos0=-1) == a(row0=4) == a(row0=-1) == a(n_new=5) == a(n_pos=0) == a(gk=None) == a(R=8) == _lib.ERR_INVALID_ARG
    del keep


def test_python_refuses():
    import modern_llm_v1_b200 as m

    x, t = torch.zeros(1, 4, 2, 64), torch.zeros(4, 32)
    y = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    call = lambda x=x, gamma=None, cos=t, y=y, rest=(1, 4, 2, 2, 64, 64): m.rotary_forward(  # noqa: E731
        x, x, cos, t, gamma, None, 1e-5, y, y, None, None, *rest)
    with pytest.raises(ValueError, match="must be CUDA"):
        call()
    with pytest.raises(ValueError, match="x must be BF16 or FP32"):
        call(x=x.half())
    with pytest.raises(ValueError, match="belong together"):
        call(gamma=torch.ones(64))
    with pytest.raises(ValueError, match="yq must be BF16"):
        call(y=y.float())
    with pytest.raises(ValueError, match="are needed"):
        call(cos=None)
    with pytest.raises(ValueError, match="scaling must be"):
        m.make_rotary_cache(8, 64, scaling="more")
    with pytest.raises(ValueError, match="trained is needed"):
        m.make_rotary_cache(8, 64, scaling="parts", factor=2.0)
    with pytest.raises(ValueError, match="even"):
        m.make_rotary_cache(8, 63)
