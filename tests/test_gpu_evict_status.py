"""Eviction by two kernels, of which the second moves what the first has listed: a unit that the first one leaves alone has no moves,
whatever the workspace held before."""
import pytest
import torch

import modern_llm_v1_b200 as m
from modern_llm_v1_b200 import _lib

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("failed", [True, False])
@pytest.mark.parametrize("L", [40, 50000])  # keys in shared memory, and too many for it
def test_moves_are_counted_for_every_unit(lib, L, failed):
    B, H, D, keep, recent = 100 if L < 100 else 40, 2, 64, 16, 4
    units, most = B * H, min(keep, L - keep)
    g = torch.Generator(device="cuda").manual_seed(L)
    k = torch.randn((B, H, L, D), generator=g, device="cuda").to(BF16)
    v, w = k.flip(2).contiguous(), torch.rand((B, H, L), generator=g, device="cuda")
    pos = torch.arange(L, dtype=I32, device="cuda").expand(B, H, L).contiguous()
    lens = torch.full((B,), L, dtype=I32, device="cuda")
    lens[::3] = 10  # nothing to be evicted
    w2, pos2 = torch.full_like(w, 3.0), torch.full_like(pos, 3)
    n = lib.b200attn_kv_evict_workspace_bytes(B, L, H, keep)
    assert n == units * (most * 8 + 4)
    ws = torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda")
    k0, v0 = k.clone(), v.clone()
    if failed:  # a position that the tables do not have
        x, y = torch.zeros((1, 1, 1, D), device="cuda"), torch.empty((1, 1, 1, D), dtype=BF16, device="cuda")
        cos, sin = m.make_rotary_cache(4, D)
        m.rotary_forward(x, x, cos, sin, None, None, 1e-5, y, y.clone(), None, None, 1, 1, 1, 1, D, D, "half", torch.tensor([[4]], dtype=I32, device="cuda"))
    rc = lib.b200attn_kv_evict(k.data_ptr(), v.data_ptr(), w.data_ptr(), pos.data_ptr(), w2.data_ptr(), pos2.data_ptr(), lens.data_ptr(), B, L, L, H, D, keep,
                               recent, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.OK
    torch.cuda.synchronize()
    moves = ws[units * most * 8:].view(I32).view(B, H)
    if failed:
        assert (moves == 0).all() and torch.equal(k, k0) and torch.equal(v, v0) and (w2 == 3).all() and (pos2 == 3).all()
        with pytest.raises(RuntimeError, match="106"):
            m.device_status()
        return
    m.device_status()
    assert (moves[::3] == 0).all()
    best = w.clone()
    best[:, :, L - recent:] = 2.0
    kept = best.topk(keep, -1).indices  # (the largest weights differ)
    assert torch.equal(moves[1::3], (kept >= keep).sum(-1).to(I32)[1::3])
    assert torch.equal(pos2[1::3, :, :keep].sort(-1).values.long(), kept.sort(-1).values[1::3])
    at = pos2[1::3, :, :keep].long()[..., None].expand(-1, -1, -1, D)
    assert torch.equal(k[1::3, :, :keep], k0[1::3].gather(2, at)) and torch.equal(v[1::3, :, :keep], v0[1::3].gather(2, at))
    assert torch.equal(k[::3], k0[::3]) and torch.equal(pos2[::3, :, :10], pos[::3, :, :10])
