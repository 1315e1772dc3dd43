"""Rotary positions of every layout against 64-bit arithmetic on the same inputs."""
import pytest
import torch

import modern_llm_v1_b200 as m
import rotary_util as ru

pytestmark = pytest.mark.gpu

EPS = 1e-5
BF16, F32 = torch.bfloat16, torch.float32
# A row's FP32 arithmetic: the rotation is three roundings of |a| + |b|, the sum of D <= 128 squares at most 128, the rest a handful:
# less than 2^-16 of the row's largest term.  BF16 results are rounded once more, by at most 2^-8 of the value.
ROW = 2.0**-16
HALF_STEP = 2.0**-8


def make(B, T, Hq, Hkv, D, R, x_type, norm, positions, x_layout, seed=0):
    g = torch.Generator().manual_seed(seed)
    xs = [torch.randn((B, H, T, D), generator=g).to(x_type) for H in (Hq, Hkv)]
    dys = [torch.randn((B, H, T, D), generator=g).to(BF16) for H in (Hq, Hkv)]
    gammas = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)] if norm else [None, None]
    n_pos = T + 37
    pos = (torch.randint(0, 37, (B, 1), generator=g) + torch.randperm(T, generator=g)[None]).to(torch.int32) if positions else None
    cos, sin = m.make_rotary_cache(n_pos, R)
    lay = (lambda t: t.transpose(1, 2).contiguous().cuda()) if x_layout == "BTHD" else (lambda t: t.contiguous().cuda())
    return xs, dys, gammas, pos, cos, sin, lay


def dev(t):
    return None if t is None else t.cuda()


def run_forward(xs, gammas, pos, cos, sin, lay, B, T, Hq, Hkv, D, R, pairs, x_layout, y_layout):
    shape = (lambda H: (B, H, T, D)) if y_layout == "BHTD" else (lambda H: (B, T, H, D))
    ys = [torch.full(shape(H), float("nan"), dtype=BF16, device="cuda") for H in (Hq, Hkv)]
    rs = [torch.full((B, H, T), float("nan"), device="cuda") if gammas[0] is not None else None for H in (Hq, Hkv)]
    m.rotary_forward(*map(lay, xs), cos, sin, *map(dev, gammas), EPS, *ys, *rs, B, T, Hq, Hkv, D, R, pairs, dev(pos), x_layout, y_layout)
    m.device_status()
    return [y if y_layout == "BHTD" else y.transpose(1, 2) for y in ys], rs


SHAPES = [  # B, T, Hq, Hkv, D, R
    (1, 1, 6, 2, 64, 64), (2, 33, 6, 2, 64, 32), (3, 17, 8, 1, 64, 16), (2, 129, 4, 4, 128, 128), (1, 70, 16, 4, 128, 96), (5, 7, 3, 3, 128, 48),
    (2, 5, 1, 1, 64, 48),
]


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("x_type,norm,positions,x_layout,y_layout", [
    (BF16, False, True, "BTHD", "BHTD"), (F32, True, False, "BTHD", "BHTD"), (F32, False, False, "BHTD", "BTHD"), (BF16, True, True, "BHTD", "BHTD"),
])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R", SHAPES)
def test_forward(B, T, Hq, Hkv, D, R, x_type, norm, positions, x_layout, y_layout, pairs):
    xs, _, gammas, pos, cos, sin, lay = make(B, T, Hq, Hkv, D, R, x_type, norm, positions, x_layout)
    ys, rs = run_forward(xs, gammas, pos, cos, sin, lay, B, T, Hq, Hkv, D, R, pairs, x_layout, y_layout)
    c, s = ru.tables(cos, sin, pos, T)
    for x, gamma, y, r in zip(xs, gammas, ys, rs):
        want, rstd = ru.forward(x.double(), None if gamma is None else gamma.double(), c, s, R, pairs, EPS)
        top = want.abs().amax(-1, keepdim=True) if gamma is None else (gamma.abs().max() * want.abs().amax(-1, keepdim=True))
        assert ((y.double().cpu() - want).abs() <= HALF_STEP * want.abs() + ROW * top).all()
        if r is not None:
            assert ((r.double().cpu() - rstd).abs() <= ROW * rstd).all()


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("x_type,norm,positions,x_layout,y_layout", [
    (BF16, False, True, "BTHD", "BHTD"), (F32, True, False, "BTHD", "BHTD"), (F32, False, False, "BHTD", "BTHD"), (BF16, True, True, "BHTD", "BHTD"),
])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R", SHAPES + [(4, 500, 6, 2, 64, 64)])
def test_backward(B, T, Hq, Hkv, D, R, x_type, norm, positions, x_layout, y_layout, pairs):
    xs, dys, gammas, pos, cos, sin, lay = make(B, T, Hq, Hkv, D, R, x_type, norm, positions, x_layout, seed=1)
    c, s = ru.tables(cos, sin, pos, T)
    leaves = [x.double().requires_grad_() for x in xs]
    gl = [None if g is None else g.double().requires_grad_() for g in gammas]
    rs = []
    for x, g, dy in zip(leaves, gl, dys):
        y, r = ru.forward(x, g, c, s, R, pairs, EPS)
        rs.append(None if r is None else r.detach().float().cuda())
        y.backward(dy.double())
    ylay = (lambda t: t.contiguous().cuda()) if y_layout == "BHTD" else (lambda t: t.transpose(1, 2).contiguous().cuda())
    dxs = [torch.full_like(lay(x), float("nan")) for x in xs]
    start = 0.25
    dgs = [None if g is None else torch.full((D,), start, device="cuda") for g in gammas]
    given = [lay(x) for x in xs] if norm else [None, None]
    m.rotary_backward(*map(ylay, dys), *given, cos, sin, *map(dev, gammas), *rs, *dxs, *dgs, B, T, Hq, Hkv, D, R, pairs, dev(pos), x_layout, y_layout)
    m.device_status()
    for x, dx, dg, leaf, g, dy in zip(xs, dxs, dgs, leaves, gl, dys):
        dx = dx.transpose(1, 2) if x_layout == "BTHD" else dx
        want = leaf.grad
        # terms of dx: rstd g and rstd^3/D s r with |s| <= sum |g r|, both below rstd max|g| (1 + sqrt(D) max|y|) with the row's rms 1/rstd
        top = dy.double().abs().amax(-1, keepdim=True)
        if g is not None:
            y, r = ru.forward(leaf.detach(), None, c, s, R, pairs, EPS)
            rstd = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
            gg = (dy.double() * g.detach()).abs()
            top = rstd * gg.amax(-1, keepdim=True) + rstd**3 / D * (gg * y.abs()).sum(-1, keepdim=True) * y.abs().amax(-1, keepdim=True)
        step = HALF_STEP if x_type == BF16 else 0.0
        assert ((dx.double().cpu() - want).abs() <= step * want.abs() + 2 * ROW * top).all()
        if g is not None:
            # a lane's rows, the warps' and the CTAs' partial sums: at most 124 additions one behind another, and four roundings of a term
            terms = (dy.double() * y * rstd).abs().sum((0, 1, 2)) + start
            assert ((dg.double().cpu() - start - g.grad).abs() <= 128 * 2.0**-24 * terms).all()


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
def test_the_gradient_is_that_of_differences(pairs):
    g = torch.Generator().manual_seed(3)
    x, gamma = torch.randn((1, 2, 3, 64), generator=g, dtype=torch.float64).requires_grad_(), torch.rand(64, generator=g, dtype=torch.float64).requires_grad_()
    a = torch.rand((1, 1, 3, 16), generator=g, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda x, w: ru.forward(x, w, a.cos(), a.sin(), 32, pairs, EPS)[0], (x, gamma))


def test_interleaved_over_the_whole_head_is_the_qknorm_operator():
    B, T, Hq, Hkv, D = 2, 100, 6, 2, 64
    xs, _, gammas, _, _, _, lay = make(B, T, Hq, Hkv, D, D, F32, True, False, "BTHD")
    cos, sin = m.make_rope_cache(T, D)
    ys, rs = run_forward(xs, gammas, None, cos, sin, lay, B, T, Hq, Hkv, D, D, "interleaved", "BTHD", "BHTD")
    yo, ro = [torch.empty_like(y) for y in ys], [torch.empty_like(r) for r in rs]
    m.rope_qknorm_forward_qk(*map(lay, xs), cos, sin, *map(dev, gammas), EPS, *yo, *ro, B, T, Hq, Hkv, D)
    for y, o, r, q in zip(ys, yo, rs, ro):
        top = o.float().abs().amax(-1, keepdim=True)  # two roundings of values that differ in the last places of FP32
        assert ((y.float() - o.float()).abs() <= 2 * HALF_STEP * o.float().abs() + 2 * ROW * top).all()
        assert ((r - q).abs() <= 2 * ROW * q).all()


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("base", 8.0), ("parts", 8.0)])
@pytest.mark.parametrize("R", [16, 64, 128])
def test_tables(scaling, factor, R):
    T, base, trained = 40000, 10000.0, 1024.0
    cos, sin = m.make_rotary_cache(T, R, base, scaling, factor, trained)
    i = torch.arange(R // 2, dtype=torch.float64)
    if scaling == "base":
        base *= factor ** (R / (R - 2))
    f = base ** (-2 * i / R)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = ((trained * f / (2 * torch.pi) - 1) / 31).clamp(0, 1)
        f = keep * f + (1 - keep) * f / factor
    angle = torch.arange(T, dtype=torch.float64)[:, None] * f
    # FP32 rounding of a value of at most one, and the angle's own rounding in 64 bits (40000 * a few 2^-52)
    for got, want in ((cos, angle.cos()), (sin, angle.sin())):
        assert (got.double().cpu() - want).abs().max() <= 2.0**-25 + 1e-9


def test_infinities_stay_in_their_pair():
    B, T, H, D, R = 1, 4, 2, 64, 32
    for pairs in ("interleaved", "half"):
        x = torch.ones((B, T, H, D), device="cuda")
        x[0, 1, 0, 40] = float("inf")  # behind the rotated part
        x[0, 2, 1, 0] = float("nan")
        cos, sin = m.make_rotary_cache(T, R)
        y = [torch.empty((B, H, T, D), dtype=BF16, device="cuda") for _ in range(2)]
        m.rotary_forward(x, x, cos, sin, None, None, EPS, *y, None, None, B, T, H, H, D, R, pairs)
        for t in y:
            bad = ~torch.isfinite(t.cpu())
            want = torch.zeros_like(bad)
            want[0, 0, 1, 40] = want[0, 1, 2, 0] = want[0, 1, 2, 1 if pairs == "interleaved" else 16] = True
            assert torch.equal(bad, want)
            assert t[0, 0, 1, 40] == float("inf")


def test_a_position_outside_the_tables_is_reported_and_its_rows_are_left():
    B, T, H, D = 2, 3, 2, 64
    x = torch.ones((B, T, H, D), device="cuda")
    cos, sin = m.make_rotary_cache(8, D)
    pos = torch.tensor([[0, 8, 2], [3, -1, 7]], dtype=torch.int32, device="cuda")
    y = [torch.full((B, H, T, D), 9.0, dtype=BF16, device="cuda") for _ in range(2)]
    m.rotary_forward(x, x, cos, sin, None, None, EPS, *y, None, None, B, T, H, H, D, D, "half", pos)
    with pytest.raises(RuntimeError, match="106"):
        m.device_status()
    m.device_status()
    for t in y:
        left = (t == 9.0).all(-1).all(1).cpu()
        assert left.tolist() == [[False, True, False], [False, True, False]]


def test_forward_attention_and_back_in_one_graph():
    """rotation, attention, its backward and the rotation back: replayed on new inputs they give what the calls give one by one"""
    B, T, Hq, Hkv, D, R = 2, 200, 6, 2, 64, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF16)  # noqa: E731
    xq, xk, v, do = new(B, T, Hq, D), new(B, T, Hkv, D), new(B, Hkv, T, D), new(B, Hq, T, D)
    cos, sin = m.make_rotary_cache(T, R, scaling="base", factor=2.0)
    e = lambda *s, dtype=BF16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    yq, yk, o, lse = e(B, Hq, T, D), e(B, Hkv, T, D), e(B, Hq, T, D), e(B, Hq, T, dtype=F32)
    dq, dk, dv, dxq, dxk = e(B, Hq, T, D), e(B, Hkv, T, D), e(B, Hkv, T, D), e(B, T, Hq, D), e(B, T, Hkv, D)

    def step():
        m.rotary_forward(xq, xk, cos, sin, None, None, EPS, yq, yk, None, None, B, T, Hq, Hkv, D, R, "half")
        m.flash_attn_forward_gqa(yq, yk, v, o, lse, B, T, Hq, Hkv, D)
        m.flash_attn_backward_gqa(yq, yk, v, o, lse, do, dq, dk, dv, B, T, Hq, Hkv, D)
        m.rotary_backward(dq, dk, None, None, cos, sin, None, None, None, None, dxq, dxk, None, None, B, T, Hq, Hkv, D, R, "half")

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    xq.copy_(new(B, T, Hq, D))
    do.copy_(new(B, Hq, T, D))
    for t in (dxq, dxk, dv):
        t.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (o, dxq, dxk, dv)]
    step()
    m.device_status()
    for a, b in zip(got, (o, dxq, dxk, dv)):
        assert torch.equal(a, b)
    # and they are the gradients of the formula
    c, s = ru.tables(cos, sin, None, T)
    q, k, vv = (t.double().cpu().requires_grad_() for t in (xq.transpose(1, 2), xk.transpose(1, 2), v))
    rq, rk = ru.rotate(q, c, s, R, "half"), ru.rotate(k, c, s, R, "half")
    a = rq @ rk.repeat_interleave(Hq // Hkv, 1).transpose(-1, -2) / D**0.5
    a = a.masked_fill(torch.ones(T, T).triu(1).bool(), -float("inf")).softmax(-1)
    (a @ vv.repeat_interleave(Hq // Hkv, 1)).backward(do.double().cpu())
    # BF16 q, k, P, dS and outputs, each 2^-8 of its value, five on the way to dx, and the sums' terms partly cancel: the parity bar
    for got_, want in ((dxq.transpose(1, 2), q.grad), (dxk.transpose(1, 2), k.grad), (dv, vv.grad)):
        d = got_.double().cpu() - want
        assert d.norm() <= 1e-2 * want.norm()
