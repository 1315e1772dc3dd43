"""Keys that hold an infinity, as BF16 leaves it of a value beyond its range."""
import math

import pytest
import torch

import modern_llm_v1_b200 as m

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("B,T,pos0,Hq,Hkv,D", [(1, 1, 20, 1, 1, 64), (2, 5, 40, 6, 2, 64), (1, 128, 0, 4, 4, 64), (1, 129, 1, 4, 2, 128),
                                               (2, 200, 55, 16, 4, 64), (1, 300, 200, 5, 1, 128), (1, 33, 100, 12, 4, 64)])
def test_a_key_that_every_token_scores_minus_infinity_weighs_nothing(B, T, pos0, Hq, Hkv, D):
    """its probability is 0 for each token, so its weight stays; the other keys' weights are those of the formula"""
    g = torch.Generator().manual_seed(T)
    J, L, scale = Hq // Hkv, pos0 + T, 1 / math.sqrt(D)
    q, k = torch.randn((B, Hq, T, D), generator=g).to(BF16), torch.randn((B, Hkv, L, D), generator=g).to(BF16)
    q[..., 3] = q[..., 3].abs() + 0.5
    far = min(L - 2, 7)
    k[:, :, far, 3] = -math.inf
    sees = torch.arange(L)[None] <= pos0 + torch.arange(T)[:, None]
    s = torch.einsum("bhjtd,bhld->bhjtl", q.double().view(B, Hkv, J, T, D), k.double()) * scale
    s = s.masked_fill(~sees, -math.inf)
    assert (s[..., far] == -math.inf).all()
    lse = s.logsumexp(-1).float()
    p = (s - lse.double()[..., None]).exp().sum((2, 3))
    w0 = torch.rand((B, Hkv, L), generator=g)
    w = w0.cuda()
    m.flash_attn_key_weights(q.cuda(), k.cuda(), lse.view(B, Hq, T).cuda(), w, B, T, pos0, Hq, Hkv, D)
    m.device_status()
    want = w0.double() + p
    # FP32 scores: D products of |q| |k| <= D * 5 * 5 at most in sum, 2^-23 of it each; exponent and sums as in the finite case
    kk = torch.where(k.isinf(), torch.zeros((), dtype=BF16), k)
    top = torch.einsum("bhtd,bhld->bhtl", q.double().abs(), kk.double().abs().repeat_interleave(J, 1)).max().item() * scale
    e = D * 2.0**-23 * top + 8 * 2.0**-24 * (top + 16)
    tol = (2 * e + 2.0**-18 + (32 + J * T / 32 + 150) * 2.0**-24) * p + 2.0**-24 * want
    assert ((w.double().cpu() - want).abs() <= tol).all()
