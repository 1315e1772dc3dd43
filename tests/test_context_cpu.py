"""What the long-context calls refuse, without a GPU."""
import ctypes

import pytest
import torch


def test_c_abi_refuses_before_any_cuda_call(lib):
    from modern_llm_v1_b200 import _lib

    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) & ~255
    s = lambda B=4, G=2, P=100, P_cap=100, L=10, L_cap=10, Hq=4, Hkv=2, D=64, q=p, ws=p, n=1 << 30: lib.b200attn_decode_shared(  # noqa: E731
        q, p, p, p, p, p, None, None, None, B, G, P, P_cap, L, L_cap, Hq, Hkv, D, 0.0, ws, n, None)
    for bad in (dict(G=3), dict(G=0), dict(P=0), dict(P_cap=99), dict(L=0), dict(L_cap=9), dict(Hkv=3), dict(q=None), dict(B=0)):
        assert s(**bad) == _lib.ERR_INVALID_ARG, bad
    assert s(D=32) == _lib.ERR_UNSUPPORTED
    assert s(q=p + 2) == _lib.ERR_ALIGNMENT
    assert s(ws=None) == s(n=100) == s(ws=p + 4) == _lib.ERR_WORKSPACE
    assert lib.b200attn_decode_shared_workspace_bytes(4, 3, 100, 10, 4, 2, 64) == 0
    w = lambda L=10, L_cap=10, Hkv=2, D=64, wt=p, ws=p, n=1 << 30, o=p: lib.b200attn_decode_weights(  # noqa: E731
        p, p, p, o, None, wt, None, 2, L, L_cap, 4, Hkv, D, 0.0, ws, n, None)
    assert w(L=0) == w(L_cap=9) == w(Hkv=3) == w(wt=None) == w(o=None) == _lib.ERR_INVALID_ARG
    assert w(D=96) == _lib.ERR_UNSUPPORTED
    assert w(o=p + 8) == _lib.ERR_ALIGNMENT
    assert w(ws=None) == w(n=64) == _lib.ERR_WORKSPACE

    c = lambda T=4, pos0=6, L_cap=10, Hkv=2, D=64, layout=0, lse=p, ws=p, n=1 << 30: lib.b200attn_key_weights(  # noqa: E731
        p, layout, p, lse, p, None, 2, T, pos0, L_cap, 4, Hkv, D, 0.0, ws, n, None)
    assert c(T=0) == c(pos0=-1) == c(pos0=7) == c(Hkv=3) == c(layout=2) == c(lse=None) == _lib.ERR_INVALID_ARG
    assert c(D=256) == _lib.ERR_UNSUPPORTED
    assert c(ws=None) == c(n=64) == _lib.ERR_WORKSPACE

    rows = 2 * 2 * 10 * 4  # bytes of an array of weights
    a = [p, p + rows, p + 2 * rows, p + 3 * rows]
    e = lambda L=10, L_cap=10, D=64, keep=4, recent=2, k=p, a=a, B=2: lib.b200attn_kv_evict(k, p, *a, None, B, L, L_cap, 2, D, keep, recent, None, 0, None)  # noqa: E731
    assert e(keep=0) == e(recent=-1) == e(recent=5) == e(L=0) == e(L_cap=9) == e(k=None) == _lib.ERR_INVALID_ARG
    assert e(D=80) == _lib.ERR_UNSUPPORTED
    assert e(k=p + 2) == _lib.ERR_ALIGNMENT
    for i, j in ((0, 2), (1, 3), (0, 3), (1, 2), (2, 3)):  # an output over an input, or over the other output
        b = list(a)
        b[j] = b[i] + 4
        assert e(a=b) == _lib.ERR_INVALID_ARG, (i, j)
    far = [p + (i << 20) for i in range(4)]
    assert e(a=far, B=100) == _lib.ERR_WORKSPACE  # 200 (batch, head) pairs: their moves are listed
    assert lib.b200attn_kv_evict_workspace_bytes(100, 10, 2, 4) == 200 * (4 * 8 + 4)
    assert lib.b200attn_kv_evict_workspace_bytes(2, 10, 2, 4) == lib.b200attn_kv_evict_workspace_bytes(100, 10, 2, 10) == 0


def test_python_refuses():
    import modern_llm_v1_b200 as m

    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    q, k, o = bf(4, 4, 64), bf(4, 2, 10, 64), bf(4, 4, 64)
    kp = bf(2, 2, 8, 64)
    with pytest.raises(ValueError, match="must be CUDA"):
        m.flash_attn_decode_shared(q, kp, kp, k, k, o, None, 4, 2, 8, 10, 4, 2, 64)
    with pytest.raises(ValueError, match="must be a tensor"):
        m.flash_attn_decode_shared(q, 3, kp, k, k, o, None, 4, 2, 8, 10, 4, 2, 64)
    with pytest.raises(ValueError, match="are needed"):
        m.flash_attn_decode_weights(q, k, k, o, None, None, 4, 10, 4, 2, 64)
    with pytest.raises(ValueError, match="weights must be FP32"):
        m.flash_attn_decode_weights(q, k, k, o, None, k, 4, 10, 4, 2, 64)
    with pytest.raises(ValueError, match="lse must be FP32"):
        m.flash_attn_key_weights(q, k, q, torch.zeros(4, 2, 10), 4, 1, 9, 4, 2, 64)
    w, p = torch.zeros(4, 2, 10), torch.zeros(4, 2, 10, dtype=torch.int32)
    with pytest.raises(ValueError, match="positions must be INT32"):
        m.kv_evict(k, k, w, p.long(), w, p, 4, 10, 2, 64, 5, 1)
    with pytest.raises(ValueError, match="must be CUDA"):
        m.kv_evict(k, k, w, p, w, p, 4, 10, 2, 64, 5, 1)


def test_kvcache_refuses():
    import modern_llm_v1_b200 as m

    new = lambda *a, **k: m.KVCache(*(a or (1, 4, 4, 2, 64, 16)), device="cpu", **k)  # noqa: E731
    for kw, what in ((dict(pairs="other"), "pairs must be"), (dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=128), "at most d_h"),
                     (dict(T_max=8), "T_max is less")):
        with pytest.raises(ValueError, match=what):
            new(**kw)
    prompts = new(1, 2, 4, 2, 64, 8)
    for a, kw, what in (((1, 3, 4, 2, 64, 8), {}, "multiple of the number"), ((2, 2, 4, 2, 64, 8), {}, "same layers"), ((1, 2, 4, 2, 64, 8), dict(T_max=64), "as theirs does"),
                        ((1, 2, 4, 2, 64, 8), dict(pairs="half"), "as theirs does"), ((1, 2, 4, 2, 64, 8), dict(track_weights=True), "keeps no weights")):
        with pytest.raises(ValueError, match=what):
            new(*a, prefix=prompts, **kw)
    c = new(1, 4, 4, 2, 64, 8, prefix=prompts)
    with pytest.raises(ValueError, match="prompts must be|same layers"):
        new(1, 4, 4, 2, 64, 8, prefix=c)
    with pytest.raises(ValueError, match="keeps no weights"):
        c.evict(4, 1)
    with pytest.raises(ValueError, match="nor behind shared"):
        c.set_lengths([1, 1, 1, 1])
    w = new(track_weights=True)
    for keep, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError, match="recent <= keep"):
            w.evict(keep, recent)
    w.evict(4, 1)  # nothing to do
    with pytest.raises(ValueError, match="new_lens"):
        w.attend(0, None, None, None, 1, new_lens=torch.ones(4))
