"""Gammas, their gradients and rstd that lie anywhere in a buffer of parameters: the bits are those of buffers of their own."""
import pytest
import torch

import modern_llm_v1_b200 as m

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("first", [1, 2, 3])
@pytest.mark.parametrize("D,R,pairs,dtype", [(64, 64, "half", BF16), (64, 32, "half", F32), (128, 96, "interleaved", BF16), (128, 128, "half", F32)])
def test_gammas_inside_a_buffer_of_parameters(D, R, pairs, dtype, first):
    B, T, Hq, Hkv = 2, 33, 6, 2
    g = torch.Generator(device="cuda").manual_seed(D + R)
    new = lambda *s, dtype=dtype: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, dy = [new(B, T, H, D) for H in (Hq, Hkv)], [new(B, H, T, D, dtype=BF16) for H in (Hq, Hkv)]
    gamma, cos, sin = [1 + 0.2 * new(D, dtype=F32) for _ in range(2)], *m.make_rotary_cache(T, R)

    def run(place):
        gm, dg = [place(t) for t in gamma], [place(torch.full((D,), 0.5, device="cuda")) for _ in range(2)]
        rstd = [place(torch.empty(B * H * T, device="cuda")) for H in (Hq, Hkv)]
        y, dx = [torch.empty_like(t) for t in dy], [torch.empty_like(t) for t in x]
        m.rotary_forward(*x, cos, sin, *gm, 1e-5, *y, *rstd, B, T, Hq, Hkv, D, R, pairs)
        m.rotary_backward(*dy, *x, cos, sin, *gm, *rstd, *dx, *dg, B, T, Hq, Hkv, D, R, pairs)
        m.device_status()
        return y + rstd + dx + dg

    def inside(t):
        buffer = torch.zeros(t.numel() + 8, device="cuda")
        part = buffer[first:first + t.numel()]
        part.copy_(t)
        assert part.data_ptr() % 16 == 4 * first
        return part

    for a, b in zip(run(lambda t: t.clone()), run(inside)):
        assert torch.equal(a, b)
