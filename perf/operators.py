"""Operators of long-context sampling, measured: rotary positions of every layout, the decode of sequences that share a prompt,
the attention weight that each cached key has received, and the eviction that goes by it.

A case is a dict of plain values.  Kinds:

  rotary_fwd, rotary_bwd  q and k of a layer rotated (part of the head, interleaved or half pairs, positions per token or the token's
                          index), with or without the QK-norm, and the way back
  shared                  one query token per sequence; G prompts, each shared by B / G sequences with caches of their own
  weights_token           one query token per sequence, and each key's probability added to its weight
  weights_chunk           the same weights for a chunk of new tokens, from the logsumexp that the forward has left
  evict                   a cache cut down to `keep` rows per head: the newest `recent`, then those of the largest weight

Shapes come from the benchmark configurations (modern-llm-v1_b200/inputs.py), the tests and ranges around them.
"""
import math

import torch

own = False  # False: plain forms in elementary torch operations; True: the package's operators

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
HEADS = ((6, 2), (16, 4), (8, 8), (12, 4), (8, 1), (4, 2))  # query heads, key/value heads
EPS = 1e-5
MAX_WORK = {"rotary": 4 * 8192 * 20 * 128, "shared": 64 * 4 * 128 * 384, "prefix": 4 * 16384 * 128, "token": 32 * 4 * 4096 * 64,
            "chunk": 16 * 4000 * 2000 * 128, "evict": 32 * 4 * 6000 * 128}


def listed():
    return [
        # one new token of one sequence, at its own position: launch latency and nothing else
        {"name": "rotary_token", "kind": "rotary_fwd", "B": 1, "T": 1, "Hq": 6, "Hkv": 2, "D": 64, "R": 64, "pairs": "half", "norm": False,
         "x": "bf16", "positions": True, "x_layout": "BTHD"},
        # a layer of the 300M-class training configuration whose projections are FP32; half of each head is rotated
        {"name": "rotary_fwd_300m", "kind": "rotary_fwd", "B": 16, "T": 1024, "Hq": 16, "Hkv": 4, "D": 64, "R": 32, "pairs": "interleaved",
         "norm": True, "x": "f32", "positions": False, "x_layout": "BTHD"},
        # the way back in the long-context training configuration, positions scaled by parts
        {"name": "rotary_bwd_long", "kind": "rotary_bwd", "B": 4, "T": 8192, "Hq": 16, "Hkv": 4, "D": 128, "R": 128, "pairs": "half",
         "norm": True, "x": "bf16", "positions": False, "x_layout": "BTHD"},
        # eight answers to one short prompt on the 50M model
        {"name": "shared_best_of_8", "kind": "shared", "B": 8, "G": 1, "P": 500, "L": 12, "Hq": 6, "Hkv": 2, "D": 64, "ragged": False},
        # sixteen answers to each of eight prompts of different lengths, some answers longer than others
        {"name": "shared_rollouts", "kind": "shared", "B": 128, "G": 8, "P": 2000, "L": 300, "Hq": 16, "Hkv": 4, "D": 64, "ragged": True},
        # many answers about one long document
        {"name": "shared_long", "kind": "shared", "B": 64, "G": 1, "P": 16384, "L": 256, "Hq": 16, "Hkv": 4, "D": 128, "ragged": False},
        # one sequence with a medium cache
        {"name": "weights_token_one", "kind": "weights_token", "B": 1, "L": 1500, "Hq": 16, "Hkv": 4, "D": 128, "ragged": False},
        # a serving batch whose sequences have different lengths
        {"name": "weights_token_batch", "kind": "weights_token", "B": 32, "L": 4096, "Hq": 16, "Hkv": 4, "D": 64, "ragged": True},
        # a long prompt, whole
        {"name": "weights_prompt", "kind": "weights_chunk", "B": 1, "T": 4000, "pos0": 0, "Hq": 16, "Hkv": 4, "D": 64},
        # a late chunk of a long prompt
        {"name": "weights_chunk", "kind": "weights_chunk", "B": 2, "T": 500, "pos0": 3000, "Hq": 16, "Hkv": 4, "D": 128},
        # one sequence that has reached the end of its cache
        {"name": "evict_one", "kind": "evict", "B": 1, "L": 2048, "keep": 1024, "recent": 256, "Hkv": 2, "D": 64, "ragged": False},
        # a batch of long caches of different lengths, cut down together
        {"name": "evict_batch", "kind": "evict", "B": 32, "L": 6000, "keep": 2500, "recent": 500, "Hkv": 4, "D": 128, "ragged": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rotary_fwd", "rotary_bwd", "shared", "shared", "weights_token", "weights_chunk", "evict"])
    Hq, Hkv = rng.choice(HEADS)
    D = rng.choice((64, 128))
    if kind.startswith("rotary"):
        B = _log(rng, 1, 32)
        x = rng.choice(("bf16", "f32"))
        T = _log(rng, 1, max(1, min(8192, MAX_WORK["rotary"] // (B * (Hq + Hkv) * D * (2 if x == "f32" else 1)))))
        R = rng.choice([r for r in (16, 32, 48, 64, 96, 128) if r <= D])
        return {"kind": kind, "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "pairs": rng.choice(("interleaved", "half")),
                "norm": rng.random() < 0.5, "x": x, "positions": rng.random() < 0.5,
                "x_layout": rng.choice(("BTHD", "BHTD"))}
    if kind == "shared":
        G, n = _log(rng, 1, 8), _log(rng, 1, 64)
        while G * n > 128:
            n -= 1
        P = _log(rng, 1, min(16384, MAX_WORK["prefix"] // (G * Hkv * D)))
        L = _log(rng, 1, min(1024, MAX_WORK["shared"] // (G * n * Hkv * D)))
        return {"kind": kind, "B": G * n, "G": G, "P": P, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "ragged": rng.random() < 0.5}
    if kind == "weights_token":
        B = _log(rng, 1, 48)
        L = _log(rng, 1, min(8192, MAX_WORK["token"] // (B * Hkv * D)))
        return {"kind": kind, "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "ragged": rng.random() < 0.5}
    if kind == "weights_chunk":
        B, T = _log(rng, 1, 8), _log(rng, 1, 4000)
        pos0 = 0 if rng.random() < 0.4 else _log(rng, 1, 4000)
        while B * Hq * T * (pos0 + T // 2) * D > MAX_WORK["chunk"]:
            T, pos0 = max(1, T // 2), pos0 // 2
        return {"kind": kind, "B": B, "T": T, "pos0": pos0, "Hq": Hq, "Hkv": Hkv, "D": D}
    B = _log(rng, 1, 32)
    L = _log(rng, 2, min(8192, MAX_WORK["evict"] // (B * Hkv * D)))
    keep = rng.randint(1, L)
    return {"kind": kind, "B": B, "L": L, "keep": keep, "recent": rng.randint(0, keep), "Hkv": Hkv, "D": D, "ragged": rng.random() < 0.5}


def _lengths(g, n, top, ragged, low=1):
    """n lengths up to `top`, one of them `top` itself"""
    if not ragged:
        return None
    lens = torch.randint(low, top + 1, (n,), generator=g, dtype=I32)
    lens[int(torch.randint(0, n, (1,), generator=g))] = top
    return lens.cuda()


def _tables(T, R):
    """cos, sin [T, R / 2]: a base of 10000 scaled by parts for contexts eight times longer than trained: pairs that turn more than 32
    times within the trained length keep their frequency, those that turn less than once have it divided, the others lie between."""
    factor, trained = 8.0, 1024.0
    i = torch.arange(R // 2, dtype=F64, device="cuda")
    freq = 10000.0 ** (-2.0 * i / R)
    turns = trained * freq / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    angle = torch.arange(T, dtype=F64, device="cuda")[:, None] * (freq * keep + freq / factor * (1.0 - keep))
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    c, s = case, {"case": case}
    g = torch.Generator().manual_seed(seed)
    gg = torch.Generator(device="cuda").manual_seed(seed + 1)
    rand = lambda *shape, dtype=BF16: torch.randn(shape, generator=gg, device="cuda").to(dtype)  # noqa: E731
    if c["kind"].startswith("rotary"):
        B, T, Hq, Hkv, D = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"]
        dt = F32 if c["x"] == "f32" else BF16
        shape = (lambda H: (B, T, H, D)) if c["x_layout"] == "BTHD" else (lambda H: (B, H, T, D))
        s["x"] = [rand(*shape(H), dtype=dt) for H in (Hq, Hkv)]
        s["gamma"] = [1 + 0.2 * rand(D, dtype=F32) for _ in range(2)] if c["norm"] else [None, None]
        # positions: every sequence of the batch begins somewhere else in the table
        s["pos"] = None
        off = torch.zeros(B, dtype=I32)
        if c["positions"]:
            off = torch.randint(0, 2048, (B,), generator=g, dtype=I32)
            s["pos"] = (off[:, None] + torch.arange(T, dtype=I32)[None]).cuda().contiguous()
        s["cos"], s["sin"] = _tables(int(off.max()) + T, c["R"])
        s["y"] = [torch.empty((B, H, T, D), dtype=BF16, device="cuda") for H in (Hq, Hkv)]
        s["rstd"] = [torch.empty((B, H, T), device="cuda") if c["norm"] else None for H in (Hq, Hkv)]
        if c["kind"] == "rotary_bwd":
            s["dy"] = [rand(B, H, T, D) for H in (Hq, Hkv)]
            s["dx"] = [torch.empty_like(x) for x in s["x"]]
            s["dg"] = [torch.zeros(D, device="cuda") if c["norm"] else None for _ in range(2)]
            if c["norm"]:  # what the forward leaves
                s["rstd"] = [torch.rsqrt(_rows(x, c).square().mean(-1) + EPS).contiguous() for x in s["x"]]
        return s
    Hkv, D, B = c["Hkv"], c["D"], c["B"]
    if c["kind"] == "shared":
        G, P, L, Hq = c["G"], c["P"], c["L"], c["Hq"]
        s["q"] = rand(B, Hq, D)
        s["kp"], s["vp"], s["k"], s["v"] = rand(G, Hkv, P, D), rand(G, Hkv, P, D), rand(B, Hkv, L, D), rand(B, Hkv, L, D)
        s["plens"], s["lens"] = _lengths(g, G, P, c["ragged"]), _lengths(g, B, L, c["ragged"])
        s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty((B, Hq), device="cuda")
        return s
    L = c["L"] if "L" in c else c["pos0"] + c["T"]
    s["k"] = rand(B, Hkv, L, D)
    s["weights"] = torch.rand((B, Hkv, L), generator=gg, device="cuda")
    if c["kind"] == "weights_token":
        Hq = c["Hq"]
        s["v"], s["q"] = rand(B, Hkv, L, D), rand(B, Hq, D)
        s["lens"] = _lengths(g, B, L, c["ragged"])
        s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty((B, Hq), device="cuda")
    elif c["kind"] == "weights_chunk":
        Hq, T = c["Hq"], c["T"]
        s["q"] = rand(B, Hq, T, D)
        s["lse"] = torch.empty((B, Hq, T), device="cuda")
        sees = torch.arange(L, device="cuda")[None] <= c["pos0"] + torch.arange(T, device="cuda")[:, None]
        for h in range(Hq):  # what the forward over the cache leaves
            sc = s["q"][:, h].float() @ s["k"][:, h // (Hq // Hkv)].float().transpose(1, 2) / math.sqrt(D)
            s["lse"][:, h] = sc.masked_fill(~sees, -math.inf).logsumexp(-1)
    else:
        s["v"] = rand(B, Hkv, L, D)
        s["lens"] = _lengths(g, B, L, c["ragged"])
        # few keys have received much of the attention, most little; some have received none and are equal
        s["weights"] = torch.relu(torch.exp(2.0 * torch.randn((B, Hkv, L), generator=gg, device="cuda")) - 0.02)
        # rows that an earlier eviction has left in some order, behind them rows in the order of their tokens
        old = min(c["keep"], L)
        pos = torch.rand((B, Hkv, old), generator=gg, device="cuda").argsort(-1)
        pos = torch.cat([pos * 2, torch.arange(2 * old, 2 * old + L - old, device="cuda").expand(B, Hkv, L - old)], -1).to(I32)
        if s["lens"] is not None:
            pos[torch.arange(L, device="cuda") >= s["lens"][:, None, None].expand(B, Hkv, 1)] = -1
        s["positions"] = pos.contiguous()
        s["weights_out"], s["positions_out"] = torch.empty_like(s["weights"]), torch.empty_like(s["positions"])
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _rows(x, c):
    """[B, H, T, D] in 32 bits"""
    x = x.float()
    return x.transpose(1, 2) if c["x_layout"] == "BTHD" else x


def _cos_sin(s, c):
    """[B or 1, 1, T, R / 2]"""
    if s["pos"] is None:
        return s["cos"][None, None, : c["T"]], s["sin"][None, None, : c["T"]]
    at = s["pos"].long()
    return s["cos"][at][:, None], s["sin"][at][:, None]


def _rotate(x, cos, sin, c):
    R = c["R"]
    out = x.clone()
    if c["pairs"] == "half":
        a, b = x[..., : R // 2], x[..., R // 2 : R]
        out[..., : R // 2], out[..., R // 2 : R] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * cos - b * sin, a * sin + b * cos
    return out


def _rotary_fwd_plain(s, c, i):
    cos, sin = _cos_sin(s, c)
    r = _rotate(_rows(s["x"][i], c), cos, sin, c)
    if not c["norm"]:
        return (r.to(BF16),)
    rstd = torch.rsqrt(r.square().mean(-1) + EPS)
    return (r * rstd[..., None] * s["gamma"][i]).to(BF16), rstd


def _rotary_bwd_plain(s, c, i):
    cos, sin = _cos_sin(s, c)
    g, extra = s["dy"][i].float(), ()
    if c["norm"]:
        r, rstd = _rotate(_rows(s["x"][i], c), cos, sin, c), s["rstd"][i][..., None]
        s["dg"][i] += (g * r * rstd).sum((0, 1, 2), dtype=F64).float()
        g = g * s["gamma"][i]
        g = rstd * g - rstd**3 * (g * r).mean(-1, keepdim=True) * r
        extra = (s["dg"][i],)
    dx = _rotate(g, cos, -sin, c)
    dx = dx.transpose(1, 2) if c["x_layout"] == "BTHD" else dx
    return (dx.to(s["x"][i].dtype).contiguous(),) + extra


def _seen(lens, L):
    """[B, 1, 1, L]: whether a row is one of the sequence's"""
    at = torch.arange(L, device="cuda")
    return (at >= 0 if lens is None else at < lens[:, None])[..., None, None, :].expand(-1 if lens is not None else 1, 1, 1, L)


def _shared_plain(s, c):
    B, G, Hq, Hkv, D = c["B"], c["G"], c["Hq"], c["Hkv"], c["D"]
    n, j = B // G, Hq // Hkv
    q = s["q"].float().view(G, n, Hkv, j, D) / math.sqrt(D)
    sp = torch.einsum("gnhjd,ghpd->gnhjp", q, s["kp"].float())
    if s["plens"] is not None:
        sp = sp.masked_fill(torch.arange(c["P"], device="cuda") >= s["plens"].view(G, 1, 1, 1, 1), -math.inf)
    so = torch.einsum("bhjd,bhld->bhjl", q.view(B, Hkv, j, D), s["k"].float())
    so = so.masked_fill(~_seen(s["lens"], c["L"]), -math.inf)
    sp = sp.reshape(B, Hkv, j, -1)
    m = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
    pp, po = (sp - m).exp(), (so - m).exp()
    z = pp.sum(-1) + po.sum(-1)
    acc = torch.einsum("gnhjp,ghpd->gnhjd", pp.reshape(G, n, Hkv, j, -1), s["vp"].float()).reshape(B, Hkv, j, D)
    acc = acc + torch.einsum("bhjl,bhld->bhjd", po, s["v"].float())
    return (acc / z[..., None]).reshape(B, Hq, D).to(BF16), (m[..., 0] + z.log()).reshape(B, Hq)


def _weights_token_plain(s, c):
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D) / math.sqrt(D)
    sc = torch.einsum("bhjd,bhld->bhjl", q, s["k"].float()).masked_fill(~_seen(s["lens"], c["L"]), -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = (sc - m).exp()
    z = p.sum(-1, keepdim=True)
    p = p / z
    s["weights"] += p.sum(2)
    o = torch.einsum("bhjl,bhld->bhjd", p, s["v"].float())
    return o.reshape(B, Hq, D).to(BF16), (m + z.log()).reshape(B, Hq), s["weights"]


def _weights_chunk_plain(s, c):
    B, T, Hq, Hkv, D, L = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"], c["pos0"] + c["T"]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, T, D) / math.sqrt(D)
    sc = torch.einsum("bhjtd,bhld->bhjtl", q, s["k"].float()) - s["lse"].view(B, Hkv, -1, T, 1)
    sees = torch.arange(L, device="cuda")[None] <= c["pos0"] + torch.arange(T, device="cuda")[:, None]
    s["weights"] += sc.masked_fill(~sees, -math.inf).exp().sum((2, 3))
    return s["weights"]


def _evict_plain(s, c):
    B, L, Hkv, D = c["B"], c["L"], c["Hkv"], c["D"]
    at = torch.arange(L, device="cuda").expand(B, Hkv, L)
    n = torch.full((B, 1, 1), L, device="cuda") if s["lens"] is None else s["lens"].view(B, 1, 1).long()
    left = n.clamp(max=c["keep"])
    live, pos = at < n, s["positions"].long()
    newest = pos.masked_fill(~live, -1).amax(-1, keepdim=True)
    key = s["weights"].masked_fill(pos > newest - c["recent"], math.inf).masked_fill(~live, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at)
    kept = rank < left
    hole, mover = (at < left) & ~kept, (at >= left) & kept
    movers = mover.to(torch.uint8).sort(dim=-1, descending=True, stable=True).indices  # the moved rows first, in their order
    src = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), at)
    rows = src[..., None].expand(B, Hkv, L, D)
    s["k"].copy_(s["k"].gather(2, rows))
    s["v"].copy_(s["v"].gather(2, rows))
    s["weights_out"].copy_(s["weights"].gather(-1, src).masked_fill(at >= left, 0.0))
    s["positions_out"].copy_(s["positions"].gather(-1, src).masked_fill(at >= left, -1))
    return s["k"], s["v"], s["weights_out"], s["positions_out"]


# ---------------------------------------------------------------------------------------------- the calls
def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "rotary_fwd":
        return _rotary_fwd_plain(s, c, 0) + _rotary_fwd_plain(s, c, 1)
    if c["kind"] == "rotary_bwd":
        return _rotary_bwd_plain(s, c, 0) + _rotary_bwd_plain(s, c, 1)
    return {"shared": _shared_plain, "weights_token": _weights_token_plain, "weights_chunk": _weights_chunk_plain, "evict": _evict_plain}[c["kind"]](s, c)


def _run_own(s, c):
    import modern_llm_v1_b200 as m

    if c["kind"].startswith("rotary"):
        dims = (c["B"], c["T"], c["Hq"], c["Hkv"], c["D"], c["R"], c["pairs"], s["pos"], c["x_layout"], "BHTD")
        if c["kind"] == "rotary_fwd":
            m.rotary_forward(*s["x"], s["cos"], s["sin"], *s["gamma"], EPS, *s["y"], *s["rstd"], *dims)
            return (s["y"][0], s["rstd"][0], s["y"][1], s["rstd"][1]) if c["norm"] else tuple(s["y"])
        m.rotary_backward(*s["dy"], *s["x"], s["cos"], s["sin"], *s["gamma"], *s["rstd"], *s["dx"], *s["dg"], *dims)
        return (s["dx"][0], s["dg"][0], s["dx"][1], s["dg"][1]) if c["norm"] else tuple(s["dx"])
    if c["kind"] == "shared":
        m.flash_attn_decode_shared(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["o"], s["lse"], c["B"], c["G"], c["P"], c["L"], c["Hq"],
                                   c["Hkv"], c["D"], s["plens"], s["lens"])
        return s["o"], s["lse"]
    if c["kind"] == "weights_token":
        m.flash_attn_decode_weights(s["q"], s["k"], s["v"], s["o"], s["lse"], s["weights"], c["B"], c["L"], c["Hq"], c["Hkv"], c["D"],
                                    s["lens"])
        return s["o"], s["lse"], s["weights"]
    if c["kind"] == "weights_chunk":
        m.flash_attn_key_weights(s["q"], s["k"], s["lse"], s["weights"], c["B"], c["T"], c["pos0"], c["Hq"], c["Hkv"], c["D"])
        return s["weights"]
    m.kv_evict(s["k"], s["v"], s["weights"], s["positions"], s["weights_out"], s["positions_out"], c["B"], c["L"], c["Hkv"], c["D"],
               c["keep"], c["recent"], s["lens"])
    return s["k"], s["v"], s["weights_out"], s["positions_out"]


# ---------------------------------------------------------------------------------------------- the least work, and 64 bits
def work(case):
    c = case
    D, Hkv, B = c["D"], c["Hkv"], c["B"]
    if c["kind"].startswith("rotary"):
        rows = B * c["T"] * (c["Hq"] + Hkv)
        x, half = 4 if c["x"] == "f32" else 2, c["T"] * c["R"] * 4  # the tables' rows, once
        if c["kind"] == "rotary_fwd":
            return {"bytes": rows * (D * (x + 2) + (4 if c["norm"] else 0)) + half, "flops": rows * (3 * c["R"] + (4 * D if c["norm"] else 0))}
        return {"bytes": rows * (D * (x + 2 + (x if c["norm"] else 0)) + (4 if c["norm"] else 0)) + half,
                "flops": rows * ((6 if c["norm"] else 3) * c["R"] + (11 * D if c["norm"] else 0))}
    mean = 0.5 if c.get("ragged") else 1.0  # of the longest
    if c["kind"] == "shared":
        G, Hq = c["G"], c["Hq"]
        keys = G * c["P"] * mean + B * c["L"] * mean
        return {"bytes": keys * Hkv * 4 * D + B * Hq * (4 * D + 4), "flops": 4 * B * Hq * D * mean * (c["P"] + c["L"])}
    if c["kind"] == "weights_token":
        keys = B * c["L"] * mean
        return {"bytes": keys * Hkv * (4 * D + 8) + B * c["Hq"] * (4 * D + 4), "flops": 4 * keys * c["Hq"] * D}
    if c["kind"] == "weights_chunk":
        T, L = c["T"], c["pos0"] + c["T"]
        pairs = T * c["pos0"] + T * (T + 1) // 2
        return {"bytes": B * (c["Hq"] * T * (2 * D + 4) + Hkv * L * (2 * D + 8)), "flops": 2 * B * c["Hq"] * pairs * D}
    L, keep, recent = c["L"], c["keep"], c["recent"]
    moved = 0.0
    for n in [L] if not c["ragged"] else [L * (k + 0.5) / 16 for k in range(16)]:
        r = min(recent, n)
        if n > keep:  # kept rows behind the first `keep`: the newest, and as many of the others as their share
            newest = min(r, n - keep)
            moved += newest + (keep - r) / max(1.0, n - r) * (n - keep - newest)
    moved *= B * Hkv / (16 if c["ragged"] else 1)
    return {"bytes": B * Hkv * L * (8 * mean + 8) + moved * 8 * D, "flops": B * Hkv * L * mean}


def exact(case, seed):
    """The same outputs from the definitions, head by head in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["kind"].startswith("rotary"):
        return _rotary_exact(s, c)
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if c["kind"] == "evict":
        return _evict_exact(s, c)
    Hq = c["Hq"]
    j, scale = Hq // Hkv, 1.0 / math.sqrt(D)
    if c["kind"] == "weights_chunk":
        T, L = c["T"], c["pos0"] + c["T"]
        w = s["weights"].double()
        for b in range(B):
            for h in range(Hq):
                a = s["q"][b, h].double().mul(scale) @ s["k"][b, h // j].double().t()
                w[b, h // j] += torch.tril(torch.exp(a - s["lse"][b, h].double()[:, None]), c["pos0"]).sum(0)
        return w
    o = torch.empty((B, Hq, D), dtype=F64, device="cuda")
    lse = torch.empty((B, Hq), dtype=F64, device="cuda")
    w = s["weights"].double() if c["kind"] == "weights_token" else None
    lens = [c["L"]] * B if s["lens"] is None else s["lens"].tolist()
    if c["kind"] == "shared":
        plens = [c["P"]] * c["G"] if s["plens"] is None else s["plens"].tolist()
    for b in range(B):
        k, v = s["k"][b, :, : lens[b]].double(), s["v"][b, :, : lens[b]].double()
        if c["kind"] == "shared":
            p = b // (B // c["G"])
            k, v = (torch.cat([a[p, :, : plens[p]].double(), x], 1) for a, x in ((s["kp"], k), (s["vp"], v)))
        a = torch.matmul(s["q"][b].double().view(Hkv, j, D), k.transpose(1, 2)) * scale
        lse[b] = torch.logsumexp(a, -1).view(Hq)
        a = torch.softmax(a, -1)
        o[b] = torch.matmul(a, v).view(Hq, D)
        if w is not None:
            w[b, :, : lens[b]] += a.sum(1)
    return (o, lse) if w is None else (o, lse, w)


def _evict_exact(s, c):
    """Head by head, with lists."""
    k, v, L = s["k"].double(), s["v"].double(), c["L"]
    w, pos = torch.zeros(s["weights"].shape, dtype=F64), torch.full(s["positions"].shape, -1, dtype=I32)
    lens = [L] * c["B"] if s["lens"] is None else s["lens"].tolist()
    for b in range(c["B"]):
        n, left = lens[b], min(lens[b], c["keep"])
        for h in range(c["Hkv"]):
            weight, at = s["weights"][b, h, :n].tolist(), s["positions"][b, h, :n].tolist()
            first = max(at) - c["recent"]
            best = sorted(range(n), key=lambda i: (at[i] <= first, 0.0 if at[i] > first else -weight[i], i))[:left]
            stays = {i for i in best if i < left}
            moves = zip([i for i in range(left) if i not in stays], sorted(i for i in best if i >= left))
            src = list(range(left))
            for to, i in moves:
                src[to] = i
            rows = torch.tensor(src, device="cuda")
            k[b, h, :left], v[b, h, :left] = k[b, h, rows], v[b, h, rows]
            w[b, h, :left], pos[b, h, :left] = torch.tensor([weight[i] for i in src], dtype=F64), torch.tensor([at[i] for i in src], dtype=I32)
    return k, v, w.cuda(), pos.cuda()


def _rotary_exact(s, c):
    """Every pair as a complex number times exp(i angle)."""
    T, R, D = c["T"], c["R"], c["D"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    turn = turn[:T].expand(c["B"], T, R // 2) if s["pos"] is None else turn[s["pos"].long()]
    turn = turn[:, None]
    one, two = (torch.arange(R // 2) * 2, torch.arange(R // 2) * 2 + 1) if c["pairs"] == "interleaved" else (torch.arange(R // 2), torch.arange(R // 2) + R // 2)
    rest = torch.arange(R, D)
    back = torch.argsort(torch.cat([one, two, rest]))

    def turned(x, by):
        z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * by
        return torch.cat([z.real, z.imag, x[..., rest]], -1)[..., back]

    out = []
    for i in range(2):
        x = s["x"][i].double()
        x = x.permute(0, 2, 1, 3) if c["x_layout"] == "BTHD" else x
        r = turned(x, turn)
        if c["kind"] == "rotary_fwd":
            if not c["norm"]:
                out.append(r)
                continue
            rstd = 1.0 / torch.sqrt(torch.sum(r * r, -1) / D + EPS)
            out += [r * rstd[..., None] * s["gamma"][i].double(), rstd]
            continue
        g = s["dy"][i].double()
        if c["norm"]:
            rstd = s["rstd"][i].double()[..., None]
            dg = torch.einsum("bhtd,bhtd,bht->d", g, r, rstd[..., 0])
            g = g * s["gamma"][i].double()
            g = rstd * (g - r * rstd**2 * torch.sum(g * r, -1, keepdim=True) / D)
        dx = turned(g, turn.conj())
        out.append(dx.permute(0, 2, 1, 3).contiguous() if c["x_layout"] == "BTHD" else dx)
        if c["norm"]:
            out.append(dg)
    return tuple(out)
