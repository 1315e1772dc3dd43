"""Decode behind shared prompts, attention weights of cached keys and eviction against 64-bit arithmetic on the same inputs.

Rows that do not count hold NaN in every test."""
import math

import pytest
import torch

import modern_llm_v1_b200 as m

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
HALF_STEP = 2.0**-8  # of a rounding to BF16
NAN = float("nan")


def randn(g, *shape, dtype=BF16):
    return torch.randn(shape, generator=g).to(dtype)


def score_error(q, k, scale):
    """What the scores of q [.., R, D] against k [.., L, D] may be off by: FP32 sums of D products, at most D 2^-23 of the sum of their
    magnitudes (a truncating adder's step), and the FP32 arithmetic of the exponent, a few 2^-24 of its size"""
    top = (q.abs() @ k.abs().transpose(-1, -2)).max().item() * scale
    return q.shape[-1] * 2.0**-23 * top + 8 * 2.0**-24 * (top + 16)


def attention(q, k, v, scale):
    """one sequence, one KV head: q [J, D], k, v [L, D] -> o, lse, p, sum p |v|, all float64"""
    s = q @ k.t() * scale
    lse = s.logsumexp(-1)
    p = (s - lse[:, None]).exp()
    return p @ v, lse, p, p @ v.abs()


def check_rows(o, lse, q, k, v, scale):
    """o [J, D] and lse [J] of the kernel against the formula"""
    wo, wl, p, mag = attention(q, k, v, scale)
    e = score_error(q, k, scale)
    # P is rounded to BF16 as the second product's operand, the result once more; the scores' error moves every p by at most 2 e
    assert ((o - wo).abs() <= HALF_STEP * wo.abs() + (HALF_STEP + 2 * e + 2.0**-14) * mag).all()
    if lse is not None:
        assert ((lse - wl).abs() <= 2 * e + 2.0**-20 * (1 + wl.abs())).all()
    return p


SHARED = [  # G, n, P, L, Hq, Hkv, D, plens, lens
    (1, 8, 500, 12, 6, 2, 64, None, None),
    (1, 1, 1, 1, 1, 1, 64, None, None),
    (1, 2, 127, 1, 4, 4, 128, None, None),
    (2, 3, 129, 65, 8, 1, 64, [0, 129], [1, 65, 2, 64, 33, 17]),
    (3, 5, 300, 70, 16, 4, 128, [300, 1, 64], None),
    (1, 64, 1000, 40, 16, 4, 64, None, None),     # 256 rows: two tiles
    (1, 50, 700, 9, 3, 1, 128, [650], None),      # 150 rows, heads that do not divide 128
    (2, 7, 2500, 300, 24, 1, 64, [2500, 1999], None),  # 24 heads of a group
    (1, 2, 260, 5, 130, 1, 64, None, None),       # more heads than a tile has rows
    (1, 16, 8200, 100, 8, 2, 128, None, None),
    (40, 2, 200, 300, 16, 4, 64, None, None),     # more tiles of rows than SMs
    (1, 4, 5000, 3000, 8, 8, 64, [4999], [3000, 1, 129, 2048]),
]


@pytest.mark.parametrize("G,n,P,L,Hq,Hkv,D,plens,lens", SHARED)
@pytest.mark.parametrize("slack", [0, 5])
def test_decode_shared(G, n, P, L, Hq, Hkv, D, plens, lens, slack):
    g = torch.Generator().manual_seed(G * 1000 + P)
    B, J, scale = G * n, Hq // Hkv, 1 / math.sqrt(D)
    q, kp, vp, k, v = randn(g, B, Hq, D), randn(g, G, Hkv, P + slack, D), randn(g, G, Hkv, P + slack, D), randn(g, B, Hkv, L + slack, D), randn(g, B, Hkv, L + slack, D)
    pl, ll = plens or [P] * G, lens or [L] * B
    for i in range(G):
        kp[i, :, pl[i]:] = vp[i, :, pl[i]:] = NAN
    for b in range(B):
        k[b, :, ll[b]:] = v[b, :, ll[b]:] = NAN
    o = torch.full((B, Hq, D), NAN, dtype=BF16, device="cuda")
    lse = torch.full((B, Hq), NAN, device="cuda")
    dev = lambda x: None if x is None else torch.tensor(x, dtype=I32, device="cuda")  # noqa: E731
    args = (B, G, P, L, Hq, Hkv, D, dev(plens), dev(lens), None, P + slack, L + slack)
    a = [t.cuda() for t in (q, kp, vp, k, v)]
    m.flash_attn_decode_shared(*a, o, lse, *args)
    m.device_status()
    oc, lc = o.double().cpu(), lse.double().cpu()
    for b in range(B):
        for h in range(Hkv):
            i, hs = b // n, slice(h * J, h * J + J)
            kk = torch.cat([kp[i, h, : pl[i]], k[b, h, : ll[b]]]).double()
            vv = torch.cat([vp[i, h, : pl[i]], v[b, h, : ll[b]]]).double()
            check_rows(oc[b, hs], lc[b, hs], q[b, hs].double(), kk, vv, scale)
    # again, without lse: the same bits
    o2 = torch.full_like(o, NAN)
    m.flash_attn_decode_shared(*a, o2, None, *args)
    assert torch.equal(o2, o)


@pytest.mark.parametrize("G,n,P,L,Hq,Hkv,D", [
    (1, 20000, 4, 2, 4, 4, 64),        # hundreds of units of a sequence's own rows for each CTA
    (64, 2, 256, 64, 16, 4, 64),       # more tiles of the prompts' rows than SMs
    (36, 16, 200, 100, 16, 4, 128),    # almost as many
    (8, 16, 2000, 300, 24, 1, 64),
    (1, 320, 200, 3500, 8, 1, 64),     # long units
    (2, 75, 900, 1, 4, 4, 128),
    (1, 12, 3220, 3, 8, 1, 128),       # few units, many splits of the prompt: clusters whose CTAs have no rows of their own
    (1, 16, 16000, 4, 8, 1, 128),
    (1, 1, 16000, 1, 4, 1, 128),
])
@pytest.mark.parametrize("ragged", [True, False])
def test_shared_prompts_of_many_sequences(G, n, P, L, Hq, Hkv, D, ragged):
    """the deals of whole units: against the formula, twice, and as a graph between whose replays other calls run"""
    g = torch.Generator(device="cuda").manual_seed(n)
    B, J, scale = G * n, Hq // Hkv, 1 / math.sqrt(D)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(BF16)

    q, kp, vp, k, v = rand(B, Hq, D), rand(G, Hkv, P, D), rand(G, Hkv, P, D), rand(B, Hkv, L, D), rand(B, Hkv, L, D)
    plens = torch.randint(0, P + 1, (G,), generator=g, device="cuda", dtype=I32)
    lens = torch.randint(1, L + 1, (B,), generator=g, device="cuda", dtype=I32) if ragged else None
    o, lse = torch.full_like(q, NAN), torch.full((B, Hq), NAN, device="cuda")

    def call(o, lse):
        m.flash_attn_decode_shared(q, kp, vp, k, v, o, lse, B, G, P, L, Hq, Hkv, D, plens, lens)

    call(o, lse)
    m.device_status()
    for b0 in range(0, B, 200):  # in float64, some sequences at a time
        b = torch.arange(b0, min(b0 + 200, B), device="cuda")
        i = b // n
        kk, vv = torch.cat([kp[i], k[b]], 2).double(), torch.cat([vp[i], v[b]], 2).double()
        qq = q[b].double().view(len(b), Hkv, J, D)
        at = torch.arange(P + L, device="cuda")
        own = (lens if ragged else torch.full((B,), L, device="cuda"))[b]
        seen = torch.where(at < P, at < plens[i, None], at - P < own[:, None])[:, None, None]
        s = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
        wl = s.logsumexp(-1)
        p = (s - wl[..., None]).exp()
        wo, mag, e = p @ vv, p @ vv.abs(), score_error(qq, kk, scale)
        err = (o[b].double().view_as(wo) - wo).abs()
        assert (err <= HALF_STEP * wo.abs() + (HALF_STEP + 2 * e + 2.0**-14) * mag).all()
        assert ((lse[b].double().view_as(wl) - wl).abs() <= 2 * e + 2.0**-20 * (1 + wl.abs())).all()
    og, lg = torch.full_like(o, NAN), torch.full_like(lse, NAN)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(og, lg)
        call(og, lg)
    for _ in range(2):
        og.fill_(NAN), lg.fill_(NAN)
        graph.replay()
        o2, l2 = torch.full_like(o, NAN), torch.full_like(lse, NAN)
        call(o2, l2)
        assert torch.equal(og, o) and torch.equal(lg, lse) and torch.equal(o2, o) and torch.equal(l2, lse)
    m.device_status()


def test_shared_prompts_with_far_apart_scores():
    """the prompt's keys outweigh the sequence's own by e^60, and the other way round"""
    G, n, P, L, H, D = 1, 4, 300, 40, 2, 64
    for big in (0, 1):
        g = torch.Generator().manual_seed(9)
        q, kp, vp, k, v = (randn(g, *s) for s in ((n, H, D), (G, H, P, D), (G, H, P, D), (n, H, L, D), (n, H, L, D)))
        q = q.abs() + 1
        (kp if big else k).mul_(0.5).add_(4)
        o, lse = torch.empty((n, H, D), dtype=BF16, device="cuda"), torch.empty((n, H), device="cuda")
        m.flash_attn_decode_shared(*(t.cuda() for t in (q, kp, vp, k, v)), o, lse, n, G, P, L, H, H, D)
        m.device_status()
        for b in range(n):
            for h in range(H):
                check_rows(o[b, h:h + 1].double().cpu(), lse[b, h:h + 1].double().cpu(), q[b, h:h + 1].double(),
                           torch.cat([kp[0, h], k[b, h]]).double(), torch.cat([vp[0, h], v[b, h]]).double(), 1 / 8)


def test_a_nan_in_the_prompt_reaches_its_sequences_only():
    G, n, P, L, H, D = 2, 2, 200, 10, 2, 64
    g = torch.Generator().manual_seed(2)
    t = [randn(g, *s).cuda() for s in ((G * n, H, D), (G, H, P, D), (G, H, P, D), (G * n, H, L, D), (G * n, H, L, D))]
    t[1][1, 0, 77, 3] = NAN
    o, lse = torch.empty((G * n, H, D), dtype=BF16, device="cuda"), torch.empty((G * n, H), device="cuda")
    m.flash_attn_decode_shared(*t, o, lse, G * n, G, P, L, H, H, D)
    m.device_status()
    bad = torch.zeros((G * n, H), dtype=torch.bool)
    bad[n:, 0] = True
    assert torch.equal(o.isnan().all(-1).cpu(), bad) and torch.equal(o.isnan().any(-1).cpu(), bad) and torch.equal(lse.isnan().cpu(), bad)


TOKEN = [  # B, L, Hq, Hkv, D, lens
    (1, 1, 1, 1, 64, None), (2, 33, 6, 2, 64, None), (1, 1500, 16, 4, 128, None), (3, 300, 5, 1, 128, [1, 300, 129]),
    (4, 700, 24, 1, 64, [699, 1, 64, 700]), (2, 64, 34, 2, 64, None), (70, 200, 8, 8, 64, None), (8, 4000, 16, 4, 64, [5, 4000, 700, 1, 2, 3, 4, 3999]),
    (2, 90, 300, 2, 64, None),
]


@pytest.mark.parametrize("B,L,Hq,Hkv,D,lens", TOKEN)
@pytest.mark.parametrize("with_lse", [True, False])
def test_decode_weights(B, L, Hq, Hkv, D, lens, with_lse):
    g = torch.Generator().manual_seed(L)
    J, cap, scale = Hq // Hkv, L + 3, 0.2
    q, k, v = randn(g, B, Hq, D), randn(g, B, Hkv, cap, D), randn(g, B, Hkv, cap, D)
    ll = lens or [L] * B
    for b in range(B):
        k[b, :, ll[b]:] = v[b, :, ll[b]:] = NAN
    w0 = torch.rand((B, Hkv, cap), generator=g) * 3
    o = torch.full((B, Hq, D), NAN, dtype=BF16, device="cuda")
    lse, w = torch.full((B, Hq), NAN, device="cuda") if with_lse else None, w0.cuda()
    m.flash_attn_decode_weights(q.cuda(), k.cuda(), v.cuda(), o, lse, w, B, L, Hq, Hkv, D,
                                None if lens is None else torch.tensor(lens, dtype=I32, device="cuda"), scale, cap)
    m.device_status()
    wc = w.double().cpu()
    for b in range(B):
        for h in range(Hkv):
            hs, n = slice(h * J, h * J + J), ll[b]
            p = check_rows(o[b, hs].double().cpu(), lse[b, hs].double().cpu() if with_lse else None, q[b, hs].double(), k[b, h, :n].double(), v[b, h, :n].double(), scale)
            e = score_error(q[b, hs].double(), k[b, h, :n].double(), scale)
            want = w0[b, h].double()
            want[:n] += p.sum(0)
            # every p is off by the score's and the lse's error, the sum by J additions
            tol = torch.full((cap,), 0.0, dtype=torch.float64)
            tol[:n] = (4 * e + 2.0**-18 + J * 2.0**-24) * p.sum(0) + 2.0**-24 * want[:n].abs()
            assert ((wc[b, h] - want).abs() <= tol).all()


CHUNK = [  # B, T, pos0, Hq, Hkv, D
    (1, 1, 0, 1, 1, 64), (2, 1, 300, 6, 2, 64), (1, 5, 1000, 8, 2, 128), (2, 33, 127, 6, 2, 64), (1, 128, 0, 4, 4, 64), (1, 129, 1, 4, 2, 128),
    (2, 200, 55, 16, 4, 64), (1, 700, 0, 12, 4, 128), (3, 500, 129, 5, 1, 64), (1, 64, 64, 24, 1, 64), (1, 1000, 2000, 6, 2, 64), (2, 3, 9, 130, 1, 64),
]


@pytest.mark.parametrize("layout", ["BHTD", "BTHD"])
@pytest.mark.parametrize("B,T,pos0,Hq,Hkv,D", CHUNK)
def test_key_weights(B, T, pos0, Hq, Hkv, D, layout):
    g = torch.Generator().manual_seed(T + pos0)
    J, L, scale = Hq // Hkv, pos0 + T, 1 / math.sqrt(D)
    cap = L + 130
    q, k = randn(g, B, Hq, T, D), randn(g, B, Hkv, cap, D)
    k[:, :, L:] = NAN
    w0 = torch.rand((B, Hkv, cap), generator=g)
    sees = torch.arange(L)[None] <= pos0 + torch.arange(T)[:, None]
    lse = torch.empty((B, Hq, T))
    want, tol = w0.double().clone(), torch.zeros((B, Hkv, cap), dtype=torch.float64)
    for b in range(B):
        for h in range(Hkv):
            s = torch.einsum("jtd,ld->jtl", q[b, h * J:h * J + J].double(), k[b, h, :L].double()) * scale
            s = s.masked_fill(~sees, -math.inf)
            lse[b, h * J:h * J + J] = s.logsumexp(-1).float()
            p = (s - lse[b, h * J:h * J + J].double()[..., None]).exp().sum((0, 1))
            want[b, h, :L] += p
            e = score_error(q[b, h * J:h * J + J].double().reshape(-1, D), k[b, h, :L].double(), scale)
            # a unit's 128 columns in four sums, then the units one behind another: at most 32 + J T / 32 additions
            tol[b, h, :L] = (2 * e + 2.0**-18 + (32 + J * T / 32 + 150) * 2.0**-24) * p + 2.0**-24 * want[b, h, :L]
    qd = (q if layout == "BHTD" else q.transpose(1, 2)).contiguous().cuda()
    w = w0.cuda()
    args = (k.cuda(), lse.cuda(), w, B, T, pos0, Hq, Hkv, D, None, cap, layout)
    m.flash_attn_key_weights(qd, *args)
    m.device_status()
    assert ((w.double().cpu() - want).abs() <= tol).all()
    first = w.clone()
    w.copy_(w0)
    m.flash_attn_key_weights(qd, *args)
    assert torch.equal(w, first)  # a call repeats bit for bit


def test_key_weights_of_a_padded_batch():
    """rows of padding, NaN in q and lse, count for nothing: every sequence's weights are those that it gets alone"""
    B, T, pos0, Hq, Hkv, D = 4, 300, 40, 4, 2, 64
    g = torch.Generator().manual_seed(7)
    q, k = randn(g, B, Hq, T, D), randn(g, B, Hkv, pos0 + T, D)
    lens = [300, 1, 130, 0]
    lse = torch.rand((B, Hq, T), generator=g) + 6
    for b, n in enumerate(lens):
        q[b, :, n:], lse[b, :, n:] = NAN, NAN
    w = torch.zeros((B, Hkv, pos0 + T), device="cuda")
    m.flash_attn_key_weights(q.cuda(), k.cuda(), lse.cuda(), w, B, T, pos0, Hq, Hkv, D, new_lens=torch.tensor(lens, dtype=I32, device="cuda"))
    for b, n in enumerate(lens):
        one = torch.zeros((1, Hkv, pos0 + T), device="cuda")
        if n:
            m.flash_attn_key_weights(q[b:b + 1, :, :n].contiguous().cuda(), k[b:b + 1].cuda(), lse[b:b + 1, :, :n].contiguous().cuda(), one, 1, n, pos0, Hq, Hkv, D,
                                     L_cap=pos0 + T)
        # the same terms in other groups: at most 32 + 2 * 300 / 32 + 150 additions each way
        assert ((w[b] - one[0]).abs() <= 2 * 201 * 2.0**-24 * one[0]).all()
    m.device_status()


def test_the_weights_of_a_prompt_are_those_of_its_tokens():
    """a prompt at once and token by token; each token hands out one unit of weight per head of the group"""
    B, T, Hq, Hkv, D = 2, 70, 6, 2, 64
    g = torch.Generator().manual_seed(4)
    q, k, v = randn(g, B, Hq, T, D).cuda(), randn(g, B, Hkv, T, D).cuda(), randn(g, B, Hkv, T, D).cuda()
    o, lse = torch.empty_like(q), torch.empty((B, Hq, T), device="cuda")
    m.flash_attn_forward_gqa(q, k, v, o, lse, B, T, Hq, Hkv, D)
    whole, single = torch.zeros((B, Hkv, T), device="cuda"), torch.zeros((B, Hkv, T), device="cuda")
    m.flash_attn_key_weights(q, k, lse, whole, B, T, 0, Hq, Hkv, D)
    ot = torch.empty((B, Hq, D), dtype=BF16, device="cuda")
    for t in range(T):
        m.flash_attn_decode_weights(q[:, :, t].contiguous(), k, v, ot, None, single, B, t + 1, Hq, Hkv, D, None, None, T)
    m.device_status()
    assert ((whole - single).abs() <= 2.0**-13 * single).all()
    assert (whole.sum(-1) - T * Hq // Hkv).abs().max() <= 2.0**-13 * T * Hq // Hkv + 1e-2


def evict_plain(k, v, w, pos, lens, keep, recent):
    """lists, one head at a time"""
    k, v = k.clone(), v.clone()
    wo, po = torch.zeros_like(w), torch.full_like(pos, -1)
    for b in range(w.shape[0]):
        n = lens[b]
        left = min(n, keep)
        for h in range(w.shape[1]):
            if n == 0:
                continue
            newest = int(pos[b, h, :n].max())
            new = [int(pos[b, h, i]) > newest - recent for i in range(n)]
            weight = [math.inf if math.isnan(x) else x for x in w[b, h, :n].tolist()]
            nan = torch.isnan(w[b, h, :n]).tolist()
            best = sorted(range(n), key=lambda i: (not new[i], (False, 0.0) if new[i] else (not nan[i], -weight[i]), i))[:left]
            free = [i for i in range(left) if i not in set(best)]
            src = list(range(left))
            for to, i in zip(free, sorted(i for i in best if i >= left)):
                src[to] = i
            k[b, h, :left], v[b, h, :left] = k[b, h, src].clone(), v[b, h, src].clone()
            wo[b, h, :left], po[b, h, :left] = w[b, h, src], pos[b, h, src]
    return k, v, wo, po


EVICT = [  # B, L, Hkv, D, keep, recent, lens, kind of weights
    (1, 1, 1, 64, 1, 0, None, "rand"), (1, 2, 1, 64, 1, 1, None, "rand"), (2, 40, 2, 64, 17, 5, [40, 3], "rand"), (1, 2048, 2, 64, 1024, 256, None, "rand"),
    (3, 300, 4, 128, 100, 0, [300, 0, 101], "ties"), (2, 600, 1, 128, 599, 599, None, "rand"), (1, 5000, 3, 64, 2500, 100, None, "zero"),
    (2, 777, 2, 64, 300, 20, None, "odd"), (70, 90, 8, 64, 30, 10, None, "rand"), (1, 9000, 1, 128, 8000, 4000, None, "ties"),
    (1, 50000, 1, 64, 20000, 500, None, "rand"), (1, 500, 2, 64, 700, 100, None, "rand"), (1, 3000, 2, 64, 1, 0, None, "ties"),
]


@pytest.mark.parametrize("B,L,Hkv,D,keep,recent,lens,kind", EVICT)
def test_evict(B, L, Hkv, D, keep, recent, lens, kind):
    g = torch.Generator().manual_seed(L + keep)
    cap = L + 4
    k, v = randn(g, B, Hkv, cap, D), randn(g, B, Hkv, cap, D)
    w = torch.rand((B, Hkv, cap), generator=g)
    if kind == "ties":
        w = (w * 7).floor()
    if kind == "zero":
        w = torch.where(w < 0.5, torch.zeros(()), -torch.zeros(()))  # 0 and -0 are equal
    if kind == "odd":
        w = torch.randn((B, Hkv, cap), generator=g) * torch.exp(20 * torch.randn((B, Hkv, cap), generator=g))
        w[:, :, 5::50], w[:, :, 7::90], w[:, :, 9::70] = NAN, math.inf, -math.inf
    pos = torch.rand((B, Hkv, cap), generator=g).argsort(-1).to(I32) * 3
    ll = lens or [L] * B
    want = evict_plain(k, v, w, pos, ll, keep, recent)
    kd, vd, wd, pd = (t.cuda() for t in (k, v, w, pos))
    wo, po = torch.full_like(wd, NAN), torch.full_like(pd, 7)
    m.kv_evict(kd, vd, wd, pd, wo, po, B, L, Hkv, D, keep, recent, None if lens is None else torch.tensor(lens, dtype=I32, device="cuda"), cap)
    m.device_status()
    assert torch.equal(po.cpu(), want[3])
    assert torch.equal(wo.cpu().view(I32), want[2].view(I32))
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
    assert torch.equal(wd.cpu().view(I32), w.view(I32)) and torch.equal(pd.cpu(), pos)


def test_attention_after_an_eviction_is_that_over_the_rows_that_stayed():
    """decode with weights, evict, decode again: the second result is the formula's over the kept set, whatever the rows' order"""
    B, L, Hq, Hkv, D, keep, recent = 2, 333, 8, 2, 64, 100, 30
    g = torch.Generator().manual_seed(8)
    q, k, v = randn(g, B, Hq, D).cuda(), randn(g, B, Hkv, L, D).cuda(), randn(g, B, Hkv, L, D).cuda()
    o, w, w2 = torch.empty_like(q), torch.zeros((B, Hkv, L), device="cuda"), torch.empty((B, Hkv, L), device="cuda")
    pos = torch.arange(L, dtype=I32, device="cuda").expand(B, Hkv, L).contiguous()
    pos2 = torch.empty_like(pos)
    m.flash_attn_decode_weights(q, k, v, o, None, w, B, L, Hq, Hkv, D)
    k0, v0 = k.clone(), v.clone()
    m.kv_evict(k, v, w, pos, w2, pos2, B, L, Hkv, D, keep, recent)
    lse = torch.empty((B, Hq), device="cuda")
    m.flash_attn_decode_weights(q, k, v, o, lse, w2, B, keep, Hq, Hkv, D, None, None, L)
    m.device_status()
    J = Hq // Hkv
    for b in range(B):
        for h in range(Hkv):
            wh = w[b, h].clone()
            wh[L - recent:] = math.inf
            kept = wh.sort(descending=True, stable=True).indices[:keep]
            assert torch.equal(pos2[b, h, :keep].sort().values.long(), kept.sort().values)
            hs = slice(h * J, h * J + J)
            check_rows(o[b, hs].double().cpu(), lse[b, hs].double().cpu(), q[b, hs].double().cpu(), k0[b, h, kept].double().cpu(), v0[b, h, kept].double().cpu(), 1 / 8)


def test_calls_in_a_graph_and_on_two_streams():
    """captured calls replayed on new inputs, and the same calls on two streams at once, give the bits of single calls"""
    B, G, P, L, Hq, Hkv, D = 16, 2, 900, 200, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF16)  # noqa: E731

    def state():
        s = dict(q=new(B, Hq, D), kp=new(G, Hkv, P, D), vp=new(G, Hkv, P, D), k=new(B, Hkv, L, D), v=new(B, Hkv, L, D))
        s.update(o=torch.empty_like(s["q"]), lse=torch.empty((B, Hq), device="cuda"), o2=torch.empty_like(s["q"]), w=torch.zeros((B, Hkv, L), device="cuda"),
                 w2=torch.empty((B, Hkv, L), device="cuda"), pos=torch.arange(L, dtype=I32, device="cuda").expand(B, Hkv, L).contiguous(),
                 pos2=torch.empty((B, Hkv, L), dtype=I32, device="cuda"), qc=new(B, Hq, 50, D), lc=torch.full((B, Hq, 50), 5.0, device="cuda"))
        return s

    def calls(s):
        s["w"].zero_()
        m.flash_attn_decode_shared(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["o"], s["lse"], B, G, P, L, Hq, Hkv, D)
        m.flash_attn_decode_weights(s["q"], s["k"], s["v"], s["o2"], None, s["w"], B, L, Hq, Hkv, D)
        m.flash_attn_key_weights(s["qc"], s["k"], s["lc"], s["w"], B, 50, L - 50, Hq, Hkv, D)
        s["kk"], s["vv"] = s["k"].clone(), s["v"].clone()
        m.kv_evict(s["kk"], s["vv"], s["w"], s["pos"], s["w2"], s["pos2"], B, L, Hkv, D, L // 2, 20)

    results = lambda s: [s[x].clone() for x in ("o", "lse", "o2", "w", "w2", "pos2", "kk", "vv")]  # noqa: E731
    states = [state() for _ in range(2)]
    want = []
    for s in states:
        calls(s)
        want.append(results(s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        for s, st in zip(states, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                calls(s)
        torch.cuda.synchronize()
        for s, w in zip(states, want):
            assert all(torch.equal(a, b) for a, b in zip(results(s), w))
    graph = torch.cuda.CUDAGraph()
    s = states[0]
    with torch.cuda.graph(graph):
        calls(s)
    for x in ("q", "kp", "vp", "k", "v", "qc"):
        s[x].copy_(states[1][x])
    for _ in range(3):
        for x in ("o", "lse", "o2", "w2"):
            s[x].fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results(s), want[1]))
    m.device_status()


def test_nothing_is_written_while_the_status_word_is_set():
    B, L, H, D = 2, 100, 2, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = randn(g, B, H, D).cuda(), randn(g, B, H, L, D).cuda(), randn(g, B, H, L, D).cuda()
    w, pos = torch.ones((B, H, L), device="cuda"), torch.arange(L, dtype=I32, device="cuda").expand(B, H, L).contiguous()
    outs = [torch.full((B, H, D), 3.0, dtype=BF16, device="cuda"), torch.full((B, H), 3.0, device="cuda"), torch.full((B, H, L), 3.0, device="cuda"),
            torch.full((B, H, L), 3, dtype=I32, device="cuda")]
    x = torch.zeros((1, 1, 1, D), device="cuda")
    cos, sin = m.make_rotary_cache(4, D)
    y = torch.empty((1, 1, 1, D), dtype=BF16, device="cuda")
    m.rotary_forward(x, x, cos, sin, None, None, 1e-5, y, y.clone(), None, None, 1, 1, 1, 1, D, D, "half", torch.tensor([[4]], dtype=I32, device="cuda"))
    k0, v0 = k.clone(), v.clone()
    m.flash_attn_decode_shared(q, k, v, k, v, outs[0], outs[1], B, B, L, L, H, H, D)
    m.flash_attn_decode_weights(q, k, v, outs[0], outs[1], w, B, L, H, H, D)
    m.flash_attn_key_weights(q.view(B, H, 1, D), k, torch.zeros((B, H, 1), device="cuda"), w, B, 1, L - 1, H, H, D)
    m.kv_evict(k, v, w, pos, outs[2], outs[3], B, L, H, D, 50, 10)
    with pytest.raises(RuntimeError, match="106"):
        m.device_status()
    assert all((t == 3).all() for t in outs) and (w == 1).all() and torch.equal(k, k0) and torch.equal(v, v0)
