"""KVCache for long contexts: other rotations, shared prompts, weights and eviction, as a sampler uses them."""
import math

import pytest
import torch

import modern_llm_v1_b200 as m
import rotary_util as ru

from gpu_util import assert_close, np32
from test_gpu_context import check_rows

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def tokens(g, B, T, Hq, Hkv, D, dtype=F32):
    new = lambda H: torch.randn((B, T, H, D), generator=g).to(dtype).cuda()  # noqa: E731
    return new(Hq), new(Hkv), new(Hkv)


def step(cache, layer, x, gammas=(None, None), new_lens=None, lse=None):
    n = x[0].shape[1]
    q = torch.full((cache.B, cache.Hq, n, cache.D), float("nan"), dtype=BF16, device="cuda")
    ctx = torch.full_like(q, float("nan"))
    lse = torch.empty((cache.B, cache.Hq, n), device="cuda") if n > 1 or lse else None
    cache.append(layer, *(t.contiguous() for t in x), *gammas, q)
    cache.attend(layer, q, ctx, lse, n, new_lens=new_lens)
    return q, ctx


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,R,pairs,scaling,dtype", [(64, 32, "half", "parts", F32), (64, 64, "half", "none", BF16), (128, 96, "interleaved", "base", F32)])
def test_rotations_of_a_cache(D, R, pairs, scaling, dtype, norm):
    """the cache holds the bits of rotary_forward, and what it attends to is the forward over them"""
    B, T, Hq, Hkv = 2, 45, 4, 2
    g = torch.Generator().manual_seed(R)
    x = tokens(g, B, T, Hq, Hkv, D, dtype)
    gammas = tuple((1 + 0.2 * torch.randn(D, generator=g)).cuda() if norm else None for _ in range(2))
    cache = m.KVCache(2, B, Hq, Hkv, D, T + 3, rotary_dim=R, pairs=pairs, scaling=scaling, factor=4.0, trained=16.0)
    cos, sin = m.make_rotary_cache(T, R, 10000.0, scaling, 4.0, 16.0)
    y = [torch.empty((B, H, T, D), dtype=BF16, device="cuda") for H in (Hq, Hkv)]
    rstd = [torch.empty((B, H, T), device="cuda") if norm else None for H in (Hq, Hkv)]
    m.rotary_forward(x[0], x[1], cos, sin, *gammas, cache.eps, *y, *rstd, B, T, Hq, Hkv, D, R, pairs)
    ctx, lse = torch.empty_like(y[0]), torch.empty((B, Hq, T), device="cuda")
    v = x[2].transpose(1, 2).to(BF16).contiguous()
    m.flash_attn_forward_gqa(y[0], y[1], v, ctx, lse, B, T, Hq, Hkv, D)
    for a, b in ((0, 20), (20, 21), (21, 43), (43, 44), (44, 45)):
        q, c = step(cache, 1, [t[:, a:b] for t in x], gammas)
        assert torch.equal(q, y[0][:, :, a:b])
        assert_close("ctx", c, np32(ctx[:, :, a:b]))
        cache.advance(b - a)
    m.device_status()
    assert torch.equal(cache.k[1, :, :, :T], y[1]) and torch.equal(cache.v[1, :, :, :T], v)
    assert cache.next_position == T
    with pytest.raises(ValueError, match="exceed the capacity"):
        step(cache, 1, [t[:, :4] for t in x], gammas)
    with pytest.raises(ValueError, match="belong together"):
        cache.append(0, *(t[:, :1].contiguous() for t in x), torch.ones(D, device="cuda"), None, q)
    with pytest.raises(ValueError, match="layer 2 out of range"):
        step(cache, 2, [t[:, :1] for t in x], gammas)


@pytest.mark.parametrize("lens", [None, [30, 7]])
@pytest.mark.parametrize("own", [False, True])
def test_sequences_that_share_prompts_are_those_that_hold_them(lens, own):
    """three samples of each of two prompts, against a cache that holds every prompt three times"""
    G, n, T, new, Hq, Hkv, D, layers = 2, 3, 30, 5, 6, 2, 64, 2
    kw = dict(rotary_dim=32, pairs="half") if own else {}
    g = torch.Generator().manual_seed(1)
    gammas = (torch.ones(D, device="cuda"), torch.ones(D, device="cuda"))
    prompts = m.KVCache(layers, G, Hq, Hkv, D, T + 2, **kw)
    whole = m.KVCache(layers, G * n, Hq, Hkv, D, T + new, **kw)
    samples = m.KVCache(layers, G * n, Hq, Hkv, D, new, prefix=prompts)
    with pytest.raises(ValueError, match="prompts are empty"):
        samples.next_position
    x = tokens(g, G, T, Hq, Hkv, D)
    for i in range(layers):
        step(prompts, i, x, gammas)
        step(whole, i, [t.repeat_interleave(n, 0) for t in x], gammas)
    prompts.advance(T)
    whole.advance(T)
    if lens:
        prompts.set_lengths(lens)
        whole.set_lengths([x for x in lens for _ in range(n)])
        prompts.k[:, 1, :, 7:] = float("nan")  # the padding's rows
        prompts.v[:, 1, :, 7:] = float("nan")
    for t in range(new):
        x = tokens(g, G * n, 1, Hq, Hkv, D)
        for i in range(layers):
            q, c = step(samples, i, x, gammas)
            qw, cw = step(whole, i, x, gammas)
            # the same positions, and rows that differ in a few last places of FP32 at most before they are rounded
            assert (q.float() - qw.float()).abs().max() <= 2.0**-6
            assert_close("ctx", c, np32(cw))
        samples.advance()
        whole.advance()
        at = samples.next_position
        assert (at == T + t + 1) if lens is None else torch.equal(at.cpu(), torch.tensor([x + t + 1 for x in lens for _ in range(n)], dtype=I32))
    m.device_status()
    with pytest.raises(ValueError, match="exceed the capacity"):
        step(samples, 0, tokens(g, G * n, 1, Hq, Hkv, D), gammas)
    prompts.reset()
    with pytest.raises(ValueError, match="prompts have changed"):
        samples.next_position
    for i in range(layers):
        step(prompts, i, tokens(g, G, T, Hq, Hkv, D), gammas)
    prompts.advance(T)
    samples.reset()
    assert samples.length == 0 and samples.next_position == T
    with pytest.raises(ValueError, match="one token per sequence"):
        step(samples, 0, tokens(g, G * n, 2, Hq, Hkv, D), gammas)


@pytest.mark.parametrize("lens", [None, [40, 9, 26]])
def test_a_sampler_that_evicts(lens):
    """prompt, tokens, eviction, tokens, eviction, tokens: every step's attention is the formula's over the rows that are left, and the
    weights are the sums of the probabilities"""
    B, T, Hq, Hkv, D, keep, recent = 3, 40, 4, 2, 64, 16, 4
    J, scale = Hq // Hkv, 1 / math.sqrt(64)
    g = torch.Generator().manual_seed(5)
    cache = m.KVCache(1, B, Hq, Hkv, D, T + 8, T_max=T + 40, rotary_dim=64, pairs="half", track_weights=True)
    cos, sin = (t.double().cpu() for t in (cache.cos, cache.sin))
    x = tokens(g, B, T, Hq, Hkv, D)
    new_lens = None if lens is None else torch.tensor(lens, dtype=I32, device="cuda")
    q, c = step(cache, 0, x, new_lens=new_lens)
    cache.advance(T)
    ll = lens or [T] * B
    if lens:
        cache.set_lengths(lens)
    held = {}  # (b, h) -> position -> [k, v, weight]
    w = cache.weights[0].double().cpu()
    kc, vc = cache.k[0].double().cpu(), cache.v[0].double().cpu()
    for b in range(B):
        for h in range(Hkv):
            s = q[b, h * J:h * J + J, : ll[b]].double().cpu() @ kc[b, h, : ll[b]].t() * scale
            s = s.masked_fill(torch.ones(ll[b], ll[b]).triu(1).bool(), -math.inf)
            p = s.softmax(-1).sum((0, 1))
            # scores and lse in FP32: 64 products of about 8 in sum, 2^-13 of a probability
            assert ((w[b, h, : ll[b]] - p).abs() <= 2.0**-13 * p).all() and (w[b, h, ll[b]:] == 0).all()
            held[b, h] = {t: [kc[b, h, t], vc[b, h, t], w[b, h, t].item()] for t in range(ll[b])}

    def check_rows_of_cache():
        n = [min(cache.length, x) for x in (cache._lengths_host or [cache.length] * B)]
        pos, k, v = cache.positions[0].cpu(), cache.k[0].double().cpu(), cache.v[0].double().cpu()
        for b in range(B):
            for h in range(Hkv):
                at = pos[b, h, : n[b]].tolist()
                assert sorted(at) == sorted(held[b, h])
                for r, t in enumerate(at):
                    assert torch.equal(k[b, h, r], held[b, h][t][0]) and torch.equal(v[b, h, r], held[b, h][t][1])
                    assert abs(cache.weights[0][b, h, r].item() - held[b, h][t][2]) <= 2.0**-12 * held[b, h][t][2]
                    held[b, h][t][2] = cache.weights[0][b, h, r].item()

    def one_token():
        x = tokens(g, B, 1, Hq, Hkv, D)
        at = cache.next_position
        at = [at] * B if isinstance(at, int) else at.tolist()
        q, c = step(cache, 0, x)
        for b in range(B):
            a = cos[at[b]], sin[at[b]]
            kk = ru.rotate(x[1][b, 0].double().cpu(), *a, 64, "half")
            qq = ru.rotate(x[0][b, 0].double().cpu(), *a, 64, "half")
            # rotated in FP32, rounded to BF16
            assert ((q[b, :, 0].double().cpu() - qq).abs() <= 2.0**-8 * qq.abs() + 2.0**-18).all()
            for h in range(Hkv):
                rows = held[b, h]
                row = (cache._lengths_host[b] if cache._lengths_host else cache.length)
                stored = cache.k[0][b, h, row].double().cpu()
                assert ((stored - kk[h]).abs() <= 2.0**-8 * kk[h].abs() + 2.0**-18).all()
                rows[at[b]] = [stored, x[2][b, 0, h].to(BF16).double().cpu(), 0.0]
                order = sorted(rows)
                ks, vs = torch.stack([rows[t][0] for t in order]), torch.stack([rows[t][1] for t in order])
                p = check_rows(c[b, h * J:h * J + J, 0].double().cpu(), None, q[b, h * J:h * J + J, 0].double().cpu(), ks, vs, scale)
                for t, add in zip(order, p.sum(0).tolist()):
                    rows[t][2] += add
        cache.advance()

    def evict():
        check_rows_of_cache()
        cache.evict(keep, recent)
        for rows in held.values():
            # (ties do not occur: the weights are sums of different probabilities)
            newest = max(rows)
            best = sorted(rows, key=lambda t: (t <= newest - recent, -rows[t][2]))[:keep]
            for t in set(rows) - set(best):
                del rows[t]
        check_rows_of_cache()

    for _ in range(3):
        one_token()
    evict()
    assert cache.length == keep
    for _ in range(7):
        one_token()
    evict()
    for _ in range(2):
        one_token()
    check_rows_of_cache()
    m.device_status()
    with pytest.raises(ValueError, match="not after an eviction"):
        cache.set_lengths([1] * B)
    cache.reset()
    assert cache.next_position == 0 and (cache.weights[0] == 0).all() and (cache.positions[0] == -1).all()


def test_positions_beyond_the_tables_are_reported():
    cache = m.KVCache(1, 1, 2, 2, 64, 8, T_max=12, track_weights=True)
    g = torch.Generator().manual_seed(0)
    x = tokens(g, 1, 8, 2, 2, 64)
    step(cache, 0, x)
    cache.advance(8)
    cache.evict(4, 2)
    step(cache, 0, [t[:, :4] for t in x])
    cache.advance(4)
    cache.evict(4, 2)
    with pytest.raises(ValueError, match="exceed the 12 positions"):
        step(cache, 0, [t[:, :1] for t in x])
    m.device_status()
