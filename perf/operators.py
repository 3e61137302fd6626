"""The token operators of tatt_amd.model.token_ops as measurable cases: attention, layer norm and rotary positions over several axes.

listed() / draw() give cases, prepare() a case's inputs on the GPU, run() one pass (the plain torch form where `own` is false, the
framework's operators where it is true), work() the bytes and operations a pass cannot do without, exact() its result in 64 bits."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5
_BASE = 10000.0


# ---- the cases --------------------------------------------------------------------------------------------------------------------
def _attention(name, direction, dtype, B, Lq, Lk, H, Hkv, D, causal=False, mask="none", layout="tokens"):
    c = {"op": "attention", "dir": direction, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D, "causal": causal,
         "mask": mask, "layout": layout}
    return {"name": name, **c} if name else c


def _norm(name, direction, dtype, R, C, residual=False, affine=True):
    c = {"op": "norm", "dir": direction, "dtype": dtype, "R": R, "C": C, "residual": residual, "affine": affine}
    return {"name": name, **c} if name else c


def _rotary(name, direction, dtype, B, T, Y, X, H, Hkv, D, s0, s1, s2, interleaved=False, far=0, layout="tokens"):
    c = {"op": "rotary", "dir": direction, "dtype": dtype, "B": B, "T": T, "Y": Y, "X": X, "H": H, "Hkv": Hkv, "D": D, "s0": s0, "s1": s1,
         "s2": s2, "interleaved": interleaved, "far": far, "layout": layout}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one image's 26 text positions through the interpreter's encoder (4 heads x 16) at inference: nothing but latency
        _attention("attn_text_positions", "forward", "fp32", 1, 26, 26, 4, 4, 16),
        # the interpreter's decoder in a training batch of 64: 1024 image tokens look at 26 text positions, words of every length
        _attention("attn_interpreter", "train", "fp32", 64, 1024, 26, 4, 4, 16, mask="lengths"),
        # self-attention of the 16x64 image tokens in fp32, the framework's default precision
        _attention("attn_image_tokens", "train", "fp32", 16, 1024, 1024, 4, 4, 64, layout="packed"),
        # self-attention over the 32x128 output map in bf16: the largest training case
        _attention("attn_output_map", "train", "bf16", 4, 4096, 4096, 8, 8, 64, layout="packed"),
        # clips, causal in time, an odd number of tokens, four query heads to a key head, padding at the end of each clip
        _attention("attn_clip_causal", "train", "bf16", 2, 2777, 2777, 16, 4, 128, causal=True, mask="lengths", layout="heads"),
        # a single new token for each of 8 sequences against the keys so far, of every length up to 20000
        _attention("attn_single_query", "forward", "bf16", 8, 1, 20000, 32, 8, 128, mask="lengths", layout="heads"),
        # the training benchmark's token matrix: 64 images x 1024 tokens x 64 channels
        _norm("norm_image_tokens", "train", "fp32", 65536, 64),
        # a wide transformer's residual stream: add and norm in one pass, bf16
        _norm("norm_wide_residual", "train", "bf16", 8192, 4096, residual=True),
        # one token of an odd width, as between two layers while serving
        _norm("norm_one_token", "forward", "bf16", 1, 1000, residual=True),
        # the 16x64 map's heads, half of the dimensions to the height and half to the width, in the training batch
        _rotary("rotary_image", "train", "fp32", 64, 1, 16, 64, 4, 4, 16, 0, 8, 8),
        # clips: time, height and width, 16 query and 4 key heads of 128, from a packed projection
        _rotary("rotary_clip", "train", "bf16", 2, 9, 32, 64, 16, 4, 128, 32, 48, 48, layout="packed"),
        # one new token for each of 32 sequences at far positions
        _rotary("rotary_far_token", "forward", "bf16", 32, 1, 1, 1, 32, 8, 128, 32, 48, 48, interleaved=True, far=1000000),
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))

    dtype = rng.choice(("fp32", "bf16"))
    op = rng.choice(("attention", "attention", "norm", "rotary"))
    if op == "attention":
        most = {"fp32": 16 * 4 * 1024 * 1024 * 64, "bf16": 4 * 8 * 4096 * 4096 * 64}[dtype]
        G, Hkv = rng.choice((1, 1, 2, 3, 4, 8)), rng.choice((1, 2, 4, 5, 8))
        D = rng.choice((16, 32, 40, 64, 64, 96, 128))
        causal, mask, layout = rng.random() < 0.4, rng.choice(("none", "lengths", "holes")), rng.choice(("tokens", "heads", "packed"))
        if rng.random() < 0.3:
            direction, Lq, Lk, layout = "forward", size(1, 4), size(1, 20000), rng.choice(("tokens", "heads"))
        else:
            direction, Lk = rng.choice(("train", "train", "forward")), size(8, 4096)  # of a few keys no gradient but rounding is left
            Lq = Lk if layout == "packed" or rng.random() < 0.5 else size(1, 4096)
        B = size(1, 64)
        while B > 1 and B * G * Hkv * Lq * Lk * D > most or B * G * Hkv * Lq * Lk > 1 << 29:
            B = max(1, B // 2)
            Hkv = max(1, Hkv - 1) if B == 1 else Hkv
            G = max(1, G - 1) if B == 1 and Hkv == 1 else G
        while G * Hkv * Lq * Lk * D > most:
            Hkv, G = (Hkv - 1, G) if Hkv > 1 else (Hkv, G - 1)
        return _attention("", direction, dtype, B, Lq, Lk, G * Hkv, Hkv, D, causal, mask, layout)
    direction = rng.choice(("train", "forward"))
    if op == "norm":
        C = size(8, 8192)  # of fewer columns the gradient is all cancellation
        R = size(1, max(1, min(65536, (1 << 25) // C)))
        return _norm("", direction, dtype, R, C, rng.random() < 0.5, rng.random() < 0.8)
    D = rng.choice((16, 32, 64, 80, 128))
    unit = D // 8
    s0, s1, s2 = rng.choice(((D, 0, 0), (0, D // 2, D // 2), (2 * unit, 3 * unit // 2 * 2, 3 * unit // 2 * 2), (2 * unit, 2 * unit, 2 * unit)))
    G, Hkv, T, Y, X = rng.choice((1, 2, 4)), rng.choice((1, 2, 4, 8)), size(1, 16), size(1, 32), size(1, 64)
    B = size(1, max(1, min(64, (1 << 26) // (T * Y * X * (G + 2) * Hkv * D))))
    while T > 1 and B * T * Y * X * (G + 2) * Hkv * D > 1 << 26:
        T = T // 2
    return _rotary("", direction, dtype, B, T, Y, X, G * Hkv, Hkv, D, s0, s1, s2, rng.random() < 0.5, rng.choice((0, 0, 1000000)),
                   rng.choice(("tokens", "heads", "packed")))


# ---- a case's inputs --------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """Visible keys of each batch element where the mask is one of lengths: spread evenly from none to all."""
    B, Lk = c["B"], c["Lk"]
    return [Lk * b // (B - 1) for b in range(B)] if B > 1 else [Lk - Lk // 4]


def _heads(layout, B, Lq, Lk, H, Hkv, D, dtype, g):
    """q [B,Lq,H,D], k and v [B,Lk,Hkv,D]: tensors of their own, head-major ones seen token-major, or slices of one projection."""
    def new(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    if layout == "packed":
        p = new(B, Lq, H + 2 * Hkv, D)
        return p[:, :, :H], p[:, :, H:H + Hkv], p[:, :, H + Hkv:]
    if layout == "heads":
        return new(B, H, Lq, D).transpose(1, 2), new(B, Hkv, Lk, D).transpose(1, 2), new(B, Hkv, Lk, D).transpose(1, 2)
    return new(B, Lq, H, D), new(B, Lk, Hkv, D), new(B, Lk, Hkv, D)


def prepare(case, seed):
    c, dtype, g = case, _TYPES[case["dtype"]], torch.Generator(device="cuda").manual_seed(int(seed))
    train = c["dir"] == "train"
    s = {"case": c, "train": train}

    def new(*shape, at=0.0, scale=1.0, as_type=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + at).to(as_type)

    def leaf(t):
        return t.detach().requires_grad_(train)

    if c["op"] == "attention":
        B, Lq, Lk, H, D = c["B"], c["Lq"], c["Lk"], c["H"], c["D"]
        q, k, v = (leaf(t) for t in _heads(c["layout"], B, Lq, Lk, H, c["Hkv"], D, dtype, g))
        s.update(q=q, k=k, v=v, causal=c["causal"], scale=D ** -0.5, mask=None, dout=new(B, Lq, H, D) if train else None)
        if c["mask"] == "lengths":
            lengths = torch.tensor(_lengths(c), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
            s["mask"] = torch.arange(Lk, device="cuda") >= lengths[:, None]
        elif c["mask"] == "holes":
            s["mask"] = torch.rand(B, Lk, generator=g, device="cuda") < 0.3
    elif c["op"] == "norm":
        R, C = c["R"], c["C"]
        s.update(x=leaf(new(R, C, at=0.3, scale=1.5)), r=leaf(new(R, C)) if c["residual"] else None, w=None, b=None,
                 dy=new(R, C) if train else None, ds=new(R, C) if train and c["residual"] else None)
        if c["affine"]:
            s.update(w=leaf(new(C, at=1.0, scale=0.2, as_type=torch.float32)), b=leaf(new(C, scale=0.2, as_type=torch.float32)))
    else:
        sections = tuple(n for n in (c["s0"], c["s1"], c["s2"]) if n)
        grid = [n for n, sec in zip((c["T"], c["Y"], c["X"]), (c["s0"], c["s1"], c["s2"])) if sec]
        B, L = c["B"], c["T"] * c["Y"] * c["X"]
        q, k, _ = _heads(c["layout"], B, L, L, c["H"], c["Hkv"], c["D"], dtype, g)
        # token l's place on each axis that has a section; sequences that go on start at places of their own
        at = torch.arange(L, device="cuda")
        strides = [math.prod(grid[i + 1:]) for i in range(len(grid))]
        positions = torch.stack([at // st % n if math.prod(grid) == L else at for st, n in zip(strides, grid)], dim=-1)
        if c["far"]:
            positions = positions + torch.randint(0, c["far"], (B, 1, len(sections)), generator=g, device="cuda")
        pairs = [torch.arange(n // 2, device="cuda", dtype=torch.float64) for n in sections]
        freqs = torch.cat([_BASE ** (-2.0 * p / n) for p, n in zip(pairs, sections)])
        s.update(q=leaf(q), k=leaf(k), positions=positions, sections=sections, freqs=freqs, interleaved=c["interleaved"],
                 dq=new(B, L, c["H"], c["D"]) if train else None, dk=new(B, L, c["Hkv"], c["D"]) if train else None)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------
def _hidden(Lq, Lk, causal, mask, device):
    """[B or 1, 1, 1, Lq or 1, Lk] truth values of the places that are left out, or None."""
    hidden = None
    if causal:
        hidden = (torch.arange(Lk, device=device) > torch.arange(Lq, device=device)[:, None] + (Lk - Lq))[None, None, None]
    if mask is not None:
        m = mask[:, None, None, None, :]
        hidden = m if hidden is None else hidden | m
    return hidden


def _plain_attention(s):
    q, k, v, dtype = s["q"].detach(), s["k"].detach(), s["v"].detach(), s["q"].dtype
    (B, Lq, H, D), Lk, Hkv = q.shape, k.shape[1], k.shape[2]
    G = H // Hkv

    def by_head(t):  # [B, L, H, D] -> fp32 [B, Hkv, G, L, D]
        return t.float().reshape(B, t.shape[1], Hkv, -1, D).permute(0, 2, 3, 1, 4).contiguous()

    def back(t, n):  # and back, rounded
        return t.permute(0, 3, 1, 2, 4).reshape(B, -1, n, D).to(dtype)

    q32, k32, v32 = by_head(q), by_head(k), by_head(v)
    p = torch.matmul(q32, k32.transpose(-1, -2)) * s["scale"]
    hidden = _hidden(Lq, Lk, s["causal"], s["mask"], q.device)
    if hidden is not None:
        p = p.masked_fill(hidden, -math.inf)
    top = p.amax(dim=-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)  # a row that sees nothing: zeros
    out = torch.matmul(p, v32)
    if not s["train"]:
        return {"out": back(out, H)}
    do = by_head(s["dout"])
    dv = torch.matmul(p.transpose(-1, -2), do).sum(dim=2, keepdim=True)
    dp = torch.matmul(do, v32.transpose(-1, -2))
    ds = p * (dp - (do * out).sum(dim=-1, keepdim=True)) * s["scale"]
    dq = torch.matmul(ds, k32)
    dk = torch.matmul(ds.transpose(-1, -2), q32).sum(dim=2, keepdim=True)
    return {"out": back(out, H), "dq": back(dq, H), "dk": back(dk, Hkv), "dv": back(dv, Hkv)}


def _plain_norm(s):
    x, dtype = s["x"].detach(), s["x"].dtype
    total = (x.float() + s["r"].detach().float()).to(dtype) if s["r"] is not None else x  # the sum is an output of the type
    t = total.float()
    t = t - t.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((t * t).mean(dim=-1, keepdim=True) + _EPS)
    xhat = t * rstd
    y = xhat * s["w"].detach() + s["b"].detach() if s["w"] is not None else xhat
    got = {"y": y.to(dtype)}
    if s["r"] is not None:
        got["sum"] = total
    if s["train"]:
        dy = s["dy"].float()
        g = dy * s["w"].detach() if s["w"] is not None else dy
        dx = rstd * (g - g.mean(dim=-1, keepdim=True) - xhat * (g * xhat).mean(dim=-1, keepdim=True))
        if s["r"] is not None:
            dx = dx + s["ds"].float()
            got["dr"] = dx.to(dtype)
        got["dx"] = dx.to(dtype)
        if s["w"] is not None:  # sums over all rows: in 64 bits
            got["dw"], got["db"] = (dy * xhat).sum(dim=0, dtype=torch.float64).float(), dy.sum(dim=0, dtype=torch.float64).float()
    return got


def _pairs(sections, interleaved, device):
    """For each pair of a head: its axis and the places of its two elements."""
    first = [sum(sections[:a]) for a in range(len(sections))]
    axis = [a for a, n in enumerate(sections) for _ in range(n // 2)]
    lo = [f + (2 * i if interleaved else i) for f, n in zip(first, sections) for i in range(n // 2)]
    hi = [f + (2 * i + 1 if interleaved else i + n // 2) for f, n in zip(first, sections) for i in range(n // 2)]
    return tuple(torch.tensor(t, device=device) for t in (axis, lo, hi))


def _turned(x, cos, sin, lo, hi):
    x32 = x.detach().float()
    u, w = x32[..., lo], x32[..., hi]
    y = x32.clone()
    y[..., lo], y[..., hi] = u * cos - w * sin, u * sin + w * cos
    return y.to(x.dtype)


def _plain_rotary(s):
    axis, lo, hi = _pairs(s["sections"], s["interleaved"], s["q"].device)
    angle = (s["positions"].double()[..., axis] * s["freqs"]).unsqueeze(-2)  # 64 bits: positions are far
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    got = {"q": _turned(s["q"], cos, sin, lo, hi), "k": _turned(s["k"], cos, sin, lo, hi)}
    if s["train"]:
        got.update(dq=_turned(s["dq"], cos, -sin, lo, hi), dk=_turned(s["dk"], cos, -sin, lo, hi))
    return got


# ---- the framework's operators ----------------------------------------------------------------------------------------------------
def _own(s):
    from tatt_amd.model import token_ops as T

    op = s["case"]["op"]
    if op == "attention":
        out = T.attention(s["q"], s["k"], s["v"], key_padding_mask=s["mask"], causal=s["causal"], scale=s["scale"])
        if not s["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if op == "norm":
        y = T.layer_norm(s["x"], s["w"], s["b"], eps=_EPS, residual=s["r"])
        got, outs, grads = {"y": y}, (y,), (s["dy"],)
        if s["r"] is not None:
            got["y"], got["sum"] = y
            outs, grads = y, (s["dy"], s["ds"])
        if s["train"]:
            leaves = {n: s[k] for n, k in (("dx", "x"), ("dr", "r"), ("dw", "w"), ("db", "b")) if s[k] is not None}
            got.update(zip(leaves, torch.autograd.grad(outs, tuple(leaves.values()), grads)))
        return got
    q, k = T.rotary(s["q"], s["k"], s["positions"], s["freqs"], s["sections"], interleaved=s["interleaved"])
    if not s["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "norm": _plain_norm, "rotary": _plain_rotary}[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    c, e, train = case, 2 if case["dtype"] == "bf16" else 4, case["dir"] == "train"
    if c["op"] == "attention":
        B, Lq, Lk, H, Hkv, D = (c[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "D"))
        lengths = _lengths(c) if c["mask"] == "lengths" else [Lk] * B
        share = 0.7 if c["mask"] == "holes" else 1.0
        if c["causal"]:
            pairs = H * sum(min(n, max(0, i + 1 + Lk - Lq)) for n in lengths for i in range(Lq)) * share
        else:
            pairs = H * Lq * sum(lengths) * share
        queries, keys = B * Lq * H * D * e, sum(lengths) * share * Hkv * D * e
        mask = B * Lk if c["mask"] != "none" else 0
        if not train:
            return {"bytes": 2 * queries + 2 * keys + mask, "flops": 4 * D * pairs}
        # reads q, k, v, dO; writes O, dq, dk, dv; two products forward, five backward
        return {"bytes": 4 * queries + 2 * keys + 2 * B * Lk * Hkv * D * e + mask, "flops": 14 * D * pairs}
    if c["op"] == "norm":
        n, res = c["R"] * c["C"], c["residual"]
        params = 8 * c["C"] if c["affine"] else 0
        if not train:
            return {"bytes": n * e * (4 if res else 2) + params, "flops": 8 * n}
        return {"bytes": n * e * (7 if res else 4) + 2 * params, "flops": 22 * n}
    n = c["B"] * c["T"] * c["Y"] * c["X"] * (c["H"] + c["Hkv"]) * c["D"]
    places = c["T"] * c["Y"] * c["X"] * (c["B"] if c["far"] else 1) * 8 * sum(bool(c[k]) for k in ("s0", "s1", "s2"))
    return {"bytes": n * e * (4 if train else 2) + places, "flops": 3 * n * (2 if train else 1)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        leaves = [s[k].detach().double().requires_grad_(s["train"]) for k in ("q", "k", "v")]
        G, Lq, Lk, outs = case["H"] // case["Hkv"], case["Lq"], case["Lk"], []
        got = {"dq": [], "dk": [], "dv": []}
        for b in range(case["B"]):  # one image or sequence at a time: 64-bit scores are large
            q, k, v = (t[b].transpose(0, 1) for t in leaves)
            scores = torch.matmul(q * s["scale"], k.repeat_interleave(G, dim=0).transpose(1, 2))
            visible = torch.ones(Lq, Lk, dtype=torch.bool, device=q.device)
            if case["causal"]:
                visible = visible.tril(Lk - Lq)
            if s["mask"] is not None:
                visible = visible & ~s["mask"][b]
            some = visible.any(dim=1, keepdim=True)
            scores = torch.where(visible, scores, torch.where(some, -math.inf, 0.0).double())
            out = torch.matmul(torch.softmax(scores, dim=-1) * some, v.repeat_interleave(G, dim=0)).transpose(0, 1)
            outs.append(out.detach())
            if s["train"]:
                for key, grad in zip(got, torch.autograd.grad(out, leaves, s["dout"][b].double())):
                    got[key].append(grad[b])
        r = {"out": torch.stack(outs)}
        if s["train"]:
            r.update({key: torch.stack(t) for key, t in got.items()})
        return r
    if case["op"] == "norm":
        x = s["x"].detach().double()
        r = {}
        if s["r"] is not None:
            r["sum"] = x + s["r"].detach().double()
            x = r["sum"].to(s["x"].dtype).double()
        x.requires_grad_(s["train"])
        w, b = (t.detach().double().requires_grad_(s["train"]) if t is not None else None for t in (s["w"], s["b"]))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + _EPS)
        y = y * w + b if w is not None else y
        r["y"] = y.detach()
        if s["train"]:
            grads = torch.autograd.grad(y, [x] + ([w, b] if w is not None else []), s["dy"].double())
            r["dx"] = grads[0] + (s["ds"].double() if s["r"] is not None else 0)
            if s["r"] is not None:
                r["dr"] = r["dx"]
            if w is not None:
                r["dw"], r["db"] = grads[1], grads[2]
        return r
    first, turns = 0, []
    for a, n in enumerate(s["sections"]):  # a section as complex numbers, each turned by its angle
        step = _BASE ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
        turns.append((first, n, torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (s["positions"][..., a, None].double() * step)).unsqueeze(-2)))
        first += n
    r = {}
    for key in ("q", "k", "dq", "dk") if s["train"] else ("q", "k"):
        x = s[key].detach().double()
        y = x.clone()
        for first, n, turn in turns:
            part = x[..., first:first + n]
            z = torch.complex(part[..., 0::2], part[..., 1::2]) if case["interleaved"] else torch.complex(part[..., :n // 2], part[..., n // 2:])
            z = z * (turn.conj() if key.startswith("d") else turn)
            y[..., first:first + n] = torch.stack((z.real, z.imag), -1).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), -1)
        r[key] = y
    return r
