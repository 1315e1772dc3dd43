"""Rows at and beyond a cache's length, given by `set_lengths` or left behind by `advance`, count as not yet written: a token that is put
there later begins without weight."""
import math

import pytest
import torch

import modern_llm_v1_b200 as m


def test_rows_beyond_the_lengths_are_cleared():
    cache = m.KVCache(2, 3, 4, 2, 64, 16, device="cpu", track_weights=True)
    for w, p in zip(cache.weights, cache.positions):
        w.copy_(torch.rand(w.shape) + 1)
        p.copy_(torch.arange(16, dtype=torch.int32).expand_as(p))
    weights, lens = [w.clone() for w in cache.weights], [0, 5, 16]
    cache.set_lengths(lens)
    for i in range(2):
        for b, n in enumerate(lens):
            assert torch.equal(cache.weights[i][b, :, :n], weights[i][b, :, :n]) and (cache.weights[i][b, :, n:] == 0).all()
            assert (cache.positions[i][b, :, :n] == torch.arange(n)).all() and (cache.positions[i][b, :, n:] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["taken back", "padding", "not accepted"])
def test_a_token_in_a_row_that_was_given_up_has_its_own_weight_only(how):
    """tokens are attended to and taken back, or a padded prompt is attended to whole, or only some of the tokens attended to are kept;
    others follow: the rows written since have the sum of the probabilities that the tokens since have given them, the rows in front
    that on top of what they had"""
    B, T, Hq, Hkv, D, cap = 3, 30, 4, 2, 64, 48
    J, scale, lens = Hq // Hkv, 1 / math.sqrt(D), {"taken back": [33, 21, 30], "padding": [30, 4, 17], "not accepted": [32, 32, 32]}[how]
    g = torch.Generator().manual_seed(3)
    ones = torch.ones(D, device="cuda")
    cache = m.KVCache(1, B, Hq, Hkv, D, cap, track_weights=True)

    def step(n, keep=None):
        x = [torch.randn((B, n, H, D), generator=g).cuda() for H in (Hq, Hkv, Hkv)]
        q, ctx = (torch.empty((B, Hq, n, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        cache.append(0, *x, ones, ones, q)
        cache.attend(0, q, ctx, torch.empty((B, Hq, n), device="cuda"), n)
        cache.advance(keep or n)
        return q

    step(T)
    if how == "taken back":
        for _ in range(3):
            step(1)
    if how == "not accepted":
        step(5, 2)
    else:
        cache.set_lengths(lens)
    want = cache.weights[0].double().cpu()
    for b, n in enumerate(lens):
        want[b, :, n:] = 0
    for t in range(4):
        q, k = step(1)[:, :, 0].double().cpu(), cache.k[0].double().cpu()
        for b in range(B):
            n = lens[b] + t + 1
            for h in range(Hkv):
                p = (q[b, h * J:h * J + J] @ k[b, h, :n].t() * scale).softmax(-1).sum(0)
                want[b, h, :n] += p
    m.device_status()
    # scores and lse in FP32: sums of 64 products of BF16 values of a norm of 8 each are off by at most 64 * 2^-23 * 8 = 2^-14, a
    # probability by twice that, in every one of the four steps
    assert ((cache.weights[0].double().cpu() - want).abs() <= 2.0**-13 * want).all()


def test_c_abi_refuses_an_append_without_weights(lib):
    from modern_llm_v1_b200 import _lib

    a = [256] * 3 + [0] + [256] * 4 + [None, None, None, 256, 256, 8, 64, 0, None, 0, None, 0, 1, 1, 4, 2, 1, 64, 1e-5, None]
    assert lib.b200attn_kv_append_weights(*a) == _lib.ERR_INVALID_ARG
