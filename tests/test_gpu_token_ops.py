"""tatt_amd.model.token_ops against plain 64-bit statements of the same operators: attention, layer norm, rotary positions, and a
transformer layer made of the three.  Bounds are elementwise and counted in roundings: a value stored in bf16 is off by at most 2^-8 of
itself (half a step), and where probabilities or score gradients enter a matrix product in bf16 every term of the sum by 2^-8 of itself;
fp32 results by a random walk of fp32 roundings along their sums (2^-15 of the sum of the terms' magnitudes: a score of 128 products has a spread of
sqrt(128) x 3 x 2^-24 = 2e-6, and 2^-15 is some fifteen times that)."""
import math

import pytest
import torch

from tatt_amd.model import token_ops as T

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
STORED = {F32: 2.0 ** -23, BF16: 2.0 ** -8}      # of the value itself
TERMS = {F32: 2.0 ** -15, BF16: 2.0 ** -8 + 2.0 ** -13}    # of the sum of the terms' magnitudes


def rnd(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def within(got, ref, terms, dtype, what, more=0.0):
    """|got - ref| <= STORED |ref| + (TERMS + more) terms, everywhere."""
    got, ref, terms = got.detach().double().cpu(), ref.detach().cpu(), terms.detach().cpu()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - (STORED[dtype] * ref.abs() + (TERMS[dtype] + more) * terms + 1e-30)
    assert over.max() <= 0 if over.numel() else True, f"{what}: over its bound by {float(over.max()):.3e} at {int(over.argmax())} (value {float(ref.flatten()[over.argmax()]):.3e})"


# ---- attention --------------------------------------------------------------------------------------------------------------------
def visible_places(B, Lq, Lk, causal, mask):
    see = torch.ones(Lq, Lk, dtype=torch.bool)
    if causal:
        see = see.tril(Lk - Lq)
    see = see[None].expand(B, Lq, Lk)
    return see & ~mask.cpu()[:, None] if mask is not None else see


def attention_64(q, k, v, do, mask, causal, scale):
    """{name: (value, sum of the terms' magnitudes)} in 64 bits on the CPU."""
    q, k, v, do = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v, do))
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    see = visible_places(B, Lq, Lk, causal, mask)[:, None]
    if mask is not None:      # what a masked key holds does not count
        k, v = (torch.where(mask.cpu()[:, None, :, None], 0.0, t) for t in (k, v))
    kh, vh = (t.repeat_interleave(H // Hk, dim=1) for t in (k, v))
    s = (q @ kh.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    lse = torch.where(see.any(-1), torch.logsumexp(s, -1), math.inf)
    p = torch.exp(s - lse[..., None]) * see
    out = p @ vh
    dp = do @ vh.transpose(2, 3)
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) * scale
    # what dS can be off by in units of TERMS: its own rounding and that of delta from the stored O and of dP
    ds_terms = p * ((dp - (do * out).sum(-1, keepdim=True)).abs() + (do * out).abs().sum(-1, keepdim=True) + (do.abs() @ vh.abs().transpose(2, 3)) * 2.0 ** -6) * abs(scale)

    def group(t):
        return t.reshape(B, Hk, H // Hk, Lk, D).sum(2)

    r = {"out": (out, p @ vh.abs()), "dq": (ds @ kh, ds_terms @ kh.abs()), "dk": (group(ds.transpose(2, 3) @ q), group(ds_terms.transpose(2, 3) @ q.abs())),
         "dv": (group(p.transpose(2, 3) @ do), group(p.transpose(2, 3) @ do.abs()))}
    r = {n: tuple(t.transpose(1, 2) for t in pair) for n, pair in r.items()}
    r["lse"] = lse
    return r


def heads(layout, B, Lq, Lk, H, Hk, D, dtype, seed):
    if layout == "packed":
        p = rnd(B, Lq, H + 2 * Hk, D, seed=seed, dtype=dtype)
        return p[:, :, :H], p[:, :, H:H + Hk], p[:, :, H + Hk:]
    if layout == "heads":
        return tuple(rnd(B, h, n, D, seed=seed + i, dtype=dtype).transpose(1, 2) for i, (h, n) in enumerate(((H, Lq), (Hk, Lk), (Hk, Lk))))
    if layout == "odd":    # rows that start at no 16-byte border
        return tuple(rnd(B, n, h, D + 1, seed=seed + i, dtype=dtype)[..., 1:] for i, (h, n) in enumerate(((H, Lq), (Hk, Lk), (Hk, Lk))))
    if layout == "apart":  # a last dimension that is not contiguous
        return tuple(rnd(B, n, D, h, seed=seed + i, dtype=dtype).transpose(2, 3) for i, (h, n) in enumerate(((H, Lq), (Hk, Lk), (Hk, Lk))))
    return tuple(rnd(B, n, h, D, seed=seed + i, dtype=dtype) for i, (h, n) in enumerate(((H, Lq), (Hk, Lk), (Hk, Lk))))


def key_mask(kind, B, Lk):
    if kind == "none":
        return None
    if kind == "lengths":   # one sequence with no key at all, one with every key
        return (torch.arange(Lk) >= torch.tensor([Lk * b // max(1, B - 1) if B > 1 else (Lk + 1) // 2 for b in range(B)])[:, None]).cuda()
    m = torch.rand(B, Lk, generator=torch.Generator().manual_seed(Lk)) < {"holes": 0.4, "most": 0.97}[kind]
    return m.cuda()


def check_attention(q, k, v, do, mask, causal, scale, what):
    ref, dtype = attention_64(q, k, v, do, mask, causal, scale), q.dtype
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = T.attention(*leaves, key_padding_mask=mask, causal=causal, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    alone, (lse, _) = T.attention_forward(q, k, v, mask, causal, scale)
    assert torch.equal(alone, out)
    with torch.no_grad():
        assert torch.equal(T.attention(q, k, v, mask, causal, scale), out)
    # the backward pass takes P from the stored lse: rounded once to fp32, it is off by at most half a step = 2^-24 of itself (in units
    # of the score), and P = exp(S - lse) by that factor: at scores of a thousand 6e-5, more than the rest of the bound
    seen = torch.isfinite(ref["lse"])
    stored_lse = 2.0 ** -24 * float(ref["lse"][seen].abs().max()) if seen.any() else 0.0
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        within(got, *ref[name], dtype, f"{what} {name}", 0.0 if name == "out" else stored_lse)
    lse, want = lse.cpu().double() * math.log(2.0), ref["lse"]
    assert torch.equal(torch.isinf(lse), torch.isinf(want)), f"{what}: empty rows"
    assert (lse - want)[seen].abs().max() <= 2.0 ** -15 * max(1.0, float(want[seen].abs().max())) if seen.any() else True, f"{what} lse"


SHAPES = [  # B, Lq, Lk, H, Hk, D
    (1, 1, 1, 1, 1, 1), (2, 1, 37, 4, 4, 16), (3, 26, 26, 4, 4, 16), (2, 300, 26, 4, 4, 16), (2, 65, 33, 2, 1, 64), (1, 130, 257, 6, 2, 40),
    (2, 33, 129, 8, 8, 128), (1, 63, 64, 3, 1, 96), (3, 128, 128, 2, 2, 32), (1, 17, 1000, 5, 1, 7), (2, 1, 3001, 8, 2, 128), (1, 3, 700, 12, 3, 64),
    (1, 1, 900, 6, 6, 120), (2, 512, 512, 2, 2, 64), (1, 257, 31, 16, 2, 128), (2, 1000, 5, 3, 3, 24)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_sizes(shape, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", B, Lq, Lk, H, Hk, D, dtype, 1)
    check_attention(q, k, v, rnd(B, Lq, H, D, seed=9, dtype=dtype), None, False, D ** -0.5, "plain")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "lengths", "holes", "most"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("shape", [(3, 70, 70, 4, 2, 64), (2, 150, 40, 2, 2, 16), (3, 40, 300, 3, 1, 128), (2, 2, 600, 8, 2, 32), (2, 333, 333, 2, 2, 40)],
                         ids=lambda s: "x".join(map(str, s)))
def test_attention_masks(shape, causal, kind, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", B, Lq, Lk, H, Hk, D, dtype, 2)
    check_attention(q, k, v, rnd(B, Lq, H, D, seed=9, dtype=dtype), key_mask(kind, B, Lk), causal, 0.3, kind)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "lengths", "front"])
@pytest.mark.parametrize("shape", [(1, 1100, 1100, 2, 2, 64), (2, 700, 1300, 4, 1, 128), (3, 1300, 600, 3, 1, 16), (1, 40, 2500, 2, 2, 96)], ids=lambda s: "x".join(map(str, s)))
def test_attention_causal_in_splits(shape, kind, dtype):
    """Long axes and few heads: every kernel splits the axis that it sums over, whose causal end differs from block to block."""
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", *shape, dtype, 3)
    mask = (torch.arange(Lk) < torch.arange(B)[:, None] * (Lk // 3) + 5).cuda() if kind == "front" else key_mask(kind, B, Lk)
    check_attention(q, k, v, rnd(B, Lq, H, D, seed=9, dtype=dtype), mask, True, D ** -0.5, kind)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["packed", "heads", "odd", "apart"])
def test_attention_layouts(layout, dtype):
    q, k, v = heads(layout, 2, 90, 90, 4, 2, 64, dtype, 3)
    do = rnd(2, 4, 90, 64, seed=9, dtype=dtype).transpose(1, 2)
    check_attention(q, k, v, do, key_mask("lengths", 2, 90), True, 0.125, layout)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_attention_broadcast_inputs(dtype):
    """Keys shared by the batch and one query for all heads (strides of 0): the gradients of the small tensors are the sums."""
    k0, v0, q0 = (rnd(*s, seed=i, dtype=dtype).requires_grad_() for i, s in enumerate(((1, 50, 2, 32), (1, 50, 2, 32), (3, 20, 1, 32))))
    do = rnd(3, 20, 4, 32, seed=5, dtype=dtype)
    out = T.attention(q0.expand(3, 20, 4, 32), k0.expand(3, 50, 2, 32), v0.expand(3, 50, 2, 32))
    got = torch.autograd.grad(out, (q0, k0, v0), do)
    ref = attention_64(q0.expand(3, 20, 4, 32), k0.expand(3, 50, 2, 32), v0.expand(3, 50, 2, 32), do, None, False, 32 ** -0.5)
    for name, g, dim in zip(("dq", "dk", "dv"), got, (2, 0, 0)):
        value, terms = (t.sum(dim, keepdim=True) for t in ref[name])
        within(g, value, terms + ref[name][0].abs().sum(dim, keepdim=True), dtype, name)   # each addend was stored, then added in the type
    within(out, *ref["out"], dtype, "out")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Lq", [1, 40])
def test_attention_masked_keys_may_hold_anything(bad, dtype, Lq):
    B, Lk, H, Hk, D = 3, 200, 4, 2, 64
    q, k, v = heads("tokens", B, Lq, Lk, H, Hk, D, dtype, 4)
    mask = key_mask("lengths", B, Lk) | key_mask("holes", B, Lk)
    do = rnd(B, Lq, H, D, seed=9, dtype=dtype)
    k[mask], v[mask] = bad, bad
    assert mask[0].all()
    check_attention(q, k, v, do, mask, False, 0.125, "garbage behind the mask")
    out, lse = T.attention_forward(q, k, v, mask)
    dq, dk, dv = T.attention_backward(do, q, k, v, out, lse, mask)
    assert not out[0].any() and not dq[0].any() and not dk[mask].any() and not dv[mask].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_attention_rows_that_see_nothing_take_no_part(dtype):
    """Causal with more queries than keys: the first rows see nothing, whatever their q and dout hold."""
    q, k, v = heads("tokens", 1, 90, 50, 4, 2, 32, dtype, 6)
    do = rnd(1, 90, 4, 32, seed=9, dtype=dtype)
    want, ref = T.attention_forward(q, k, v, causal=True), None
    ref = T.attention_backward(do, q, k, v, *want, causal=True)
    do[:, :40], q[:, :40] = float("nan"), float("inf")
    out, lse = T.attention_forward(q, k, v, causal=True)
    got = T.attention_backward(do, q, k, v, out, lse, causal=True)
    assert torch.equal(out, want[0]) and not out[:, :40].any() and torch.isinf(lse[0][:, :, :40]).all()
    assert not got[0][:, :40].any()
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 90, 90, 4, 2, 32), (2, 40, 300, 4, 4, 128), (2, 600, 20, 2, 1, 64)], ids=lambda s: "x".join(map(str, s)))
def test_attention_rows_that_see_only_masked_keys_take_no_part(shape, dtype):
    """Causal with padding in front: the first rows see masked keys alone, whatever their q and dout hold."""
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", *shape, dtype, 6)
    do = rnd(B, Lq, H, D, seed=9, dtype=dtype)
    first = Lk - Lq + 30 if Lk > 30 else 10           # the first key that is not masked; row 0 sees Lk - Lq + 1 keys
    mask = (torch.arange(Lk) < torch.tensor([[first], [0]])).cuda()
    blind = first - (Lk - Lq)                         # rows of the first sequence that see nothing
    want = T.attention_forward(q, k, v, mask, True)
    ref = T.attention_backward(do, q, k, v, *want, mask, True)
    do[0, :blind], q[0, :blind] = float("nan"), float("inf")
    out, saved = T.attention_forward(q, k, v, mask, True)
    got = T.attention_backward(do, q, k, v, out, saved, mask, True)
    assert torch.equal(out, want[0]) and not out[0, :blind].any() and torch.isinf(saved[0][0, :, :blind]).all() and torch.isfinite(saved[0][0, :, blind:]).all()
    assert not got[0][0, :blind].any()
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [1, 70])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [5e3, 1e16])
def test_attention_scores_far_from_zero(dtype, Lq, sign, size):
    """Scores whose steps are too large for more than one key: up to 2^29 the choice of that key; past it NaN, never a row of zeros."""
    k = (torch.linspace(2, 1, 40) * sign * size).to(dtype).cuda()[None, :, None, None].expand(2, 40, 2, 16)
    q, v = torch.full((2, Lq, 2, 16), size, dtype=dtype, device="cuda"), rnd(2, 40, 2, 16, seed=1, dtype=dtype)
    out, saved = T.attention_forward(q, k, v)
    if size == 1e16:
        assert torch.isnan(out).all() and torch.isnan(saved[0]).all()
        assert all(torch.isnan(g).all() for g in T.attention_backward(torch.ones_like(q), q, k, v, out, saved))
        return
    pick = v[:, 0 if sign > 0 else 39][:, None].expand_as(out).double().cpu()
    within(out, pick, pick.abs(), dtype, "the chosen value")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("scale", [40.0, 0.0, -0.25])
def test_attention_large_and_odd_scales(scale, dtype):
    """Scores of some hundreds: the softmax is nearly a choice of one key; 0: the mean of the values; negative: the other way round."""
    q, k, v = heads("tokens", 2, 50, 120, 2, 2, 32, dtype, 7)
    if scale == 40.0:
        q, k = q.sign(), k.sign()       # whole scores: products and sums are exact in both types, neighbours 80 apart
        do = rnd(2, 50, 2, 32, seed=9, dtype=dtype)
        check_attention(q, k, v, do, None, False, scale, "large")
    else:
        check_attention(q, k, v, rnd(2, 50, 2, 32, seed=9, dtype=dtype), None, True, scale, "scale")


def test_attention_gradient_against_differences():
    q, k, v = (t.double().float() for t in heads("tokens", 2, 40, 70, 4, 2, 32, F32, 8))
    mask, w = key_mask("holes", 2, 70), rnd(2, 40, 4, 32, seed=10)
    out, lse = T.attention_forward(q, k, v, mask, True)
    grads = T.attention_backward(w, q, k, v, out, lse, mask, True)

    def value(*t):
        return float((T.attention(*t, key_padding_mask=mask, causal=True).double() * w.double()).sum())

    for i in range(3):   # steps of h: the error is of order h^2 and of 2^-24 |values| / h, both some 1e-4 of the slope at h = 2^-7
        d = rnd(*(q, k, v)[i].shape, seed=20 + i)
        h = 2.0 ** -7
        at = [[t + sgn * h * d if j == i else t for j, t in enumerate((q, k, v))] for sgn in (1, -1)]
        slope, want = (value(*at[0]) - value(*at[1])) / (2 * h), float((grads[i].double() * d.double()).sum())
        size = float(grads[i].double().norm() * d.double().norm())
        assert abs(slope - want) <= 1e-3 * size, (i, slope, want)


def test_attention_offsets_past_32_bits():
    """Two sequences whose keys lie more than 2^31 elements apart."""
    far, L, Hk, D = (1 << 31) + 4096, 70, 2, 64
    big = torch.empty(far + L * Hk * D, dtype=BF16, device="cuda")
    k = big.as_strided((2, L, Hk, D), (far, Hk * D, D, 1))
    k.copy_(rnd(2, L, Hk, D, seed=1, dtype=BF16))
    q, v, do = (rnd(2, n, h, D, seed=2 + n, dtype=BF16) for n, h in ((33, 4), (L, Hk), (33, 4)))
    check_attention(q, k, v, do, None, False, 0.125, "far keys")
    check_attention(q[:, :1], k, v, do[:, :1], None, False, 0.125, "far keys, one query")


@pytest.mark.parametrize("dims", [(0, 4, 5), (2, 0, 5), (2, 4, 0)])
def test_attention_of_nothing(dims):
    B, Lq, Lk = dims
    q, k, v = (torch.randn(B, n, 2, 16, device="cuda", requires_grad=True) for n in (Lq, Lk, Lk))
    out = T.attention(q, k, v)
    assert out.shape == q.shape and not out.any()
    for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 1, 5000, 8, 2, 128), (2, 1024, 26, 4, 4, 16), (1, 700, 700, 4, 4, 64)], ids=lambda s: "x".join(map(str, s)))
def test_attention_is_reproducible_on_any_stream(shape, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", B, Lq, Lk, H, Hk, D, dtype, 11)
    do = rnd(B, Lq, H, D, seed=9, dtype=dtype)

    def both():
        out, lse = T.attention_forward(q, k, v)
        return (out, *(t for t in lse if t is not None), *T.attention_backward(do, q, k, v, out, lse))

    want, streams, got = both(), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams * 2:      # two calls in flight at once: each has a workspace of its own
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


# ---- layer norm -------------------------------------------------------------------------------------------------------------------
def norm_64(s, w, b, dy, ds, eps):
    s, dy = s.detach().cpu().double(), dy.cpu().double()
    w, b = (t.detach().cpu().double() if t is not None else None for t in (w, b))
    mu = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mu) ** 2).mean(-1, keepdim=True) + eps)
    xhat = (s - mu) * rstd
    g = dy * w if w is not None else dy
    y = xhat * (1 if w is None else w) + (0 if b is None else b)
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    ds = 0 if ds is None else ds.cpu().double()
    # magnitudes of what is added: a mean's error is a rounding of its largest terms
    big = s.abs().amax(-1, keepdim=True) * rstd
    y_terms = (big + xhat.abs()) * (1 if w is None else w.abs()) + (0 if b is None else b.abs())
    hs = 1 + big
    dx_terms = rstd * hs * (g.abs() + g.abs().amax(-1, keepdim=True) * (1 + xhat.abs()))
    rows = tuple(range(s.dim() - 1))
    return {"y": (y, y_terms), "dx": (dx + ds, dx_terms + (ds.abs() if torch.is_tensor(ds) else 0)), "dw": ((dy * xhat).sum(rows), (dy.abs() * (xhat.abs() + big)).sum(rows)),
            "db": (dy.sum(rows), dy.abs().sum(rows))}


def within_norm(got, pair, dtype, what):
    """y and dx leave in `dtype`, everything before is fp32: a few fp32 roundings of the terms, then the stored one."""
    got, (ref, terms) = got.detach().double().cpu(), pair
    bound = STORED[dtype] * ref.abs() + 2.0 ** -20 * terms + 1e-30     # sixteen fp32 roundings of the largest term
    assert torch.isfinite(got).all(), what
    assert ((got - ref).abs() <= bound).all(), f"{what}: {float(((got - ref).abs() - bound).max()):.3e} over"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("R,C", [(1, 1), (5, 2), (1, 1000), (130, 7), (1664, 64), (3, 64), (513, 100), (2000, 128), (77, 777), (300, 1024), (33, 2048), (19, 4096),
                                 (9, 8200), (3, 20001), (70000, 8)])
def test_layer_norm(R, C, residual, dtype):
    x, r = rnd(R, C, seed=1, dtype=dtype, scale=2.0) + 0.5, rnd(R, C, seed=2, dtype=dtype)
    w, b = rnd(C, seed=3) * 0.3 + 1, rnd(C, seed=4)
    dy, ds = rnd(R, C, seed=5, dtype=dtype), rnd(R, C, seed=6, dtype=dtype)
    leaves = [t.requires_grad_() for t in ((x, r, w, b) if residual else (x, w, b))]
    got = T.layer_norm(x, w, b, residual=r if residual else None)
    if residual:
        y, s = got
        assert torch.equal(s, (x.float() + r.float()).to(dtype))
        grads = torch.autograd.grad((y, s), leaves, (dy, ds))
        assert torch.equal(grads[0], grads[1])
    else:
        y, s = got, x
        grads = torch.autograd.grad(y, leaves, dy)
    ref = norm_64(s, w, b, dy, ds if residual else None, 1e-5)
    for name, g in zip(("y", "dx", "dw", "db"), (y, grads[0], grads[-2], grads[-1])):
        within_norm(g, ref[name], dtype if name in ("y", "dx") else F32, name)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("C", [64, 100, 1001])
def test_layer_norm_layouts(C, dtype):
    """Rows further apart than their width and at no 16-byte border; leading dimensions; without weight, without bias, without either."""
    wide = rnd(50, C + 3, seed=1, dtype=dtype)
    w, dy = rnd(C, seed=3) + 1, rnd(50, C + 5, seed=5, dtype=dtype)[:, 2:2 + C]
    for x in (wide[:, 3:], wide[:, :C], rnd(5, 10, C, seed=7, dtype=dtype), rnd(C, 50, seed=7, dtype=dtype).t(), rnd(1, C, seed=7, dtype=dtype).expand(50, C)):
        for weight, bias in ((w, None), (None, w), (None, None)):
            d = dy.reshape(x.shape)
            y, s, stat = T.layer_norm_forward(x, weight, bias)
            ds, dw, db = T.layer_norm_backward(d, s, weight, stat)
            ref = norm_64(x, weight, bias, d, None, 1e-5)
            for name, g in (("y", y), ("dx", ds), ("dw", dw), ("db", db)):
                within_norm(g, ref[name], dtype if name in ("y", "dx") else F32, name)


def test_layer_norm_one_output_used_and_rows_of_one_value():
    x, r = (rnd(6, 40, seed=i).requires_grad_() for i in (1, 2))
    w = rnd(40, seed=3).requires_grad_()
    y, s = T.layer_norm(x, w, residual=r)
    a, b = torch.autograd.grad(s.sum(), (x, r), retain_graph=True)
    assert torch.equal(a, torch.ones_like(a)) and torch.equal(b, a)
    gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    ref = norm_64(s, w, None, torch.ones_like(y), None, 1e-5)
    within_norm(gx, ref["dx"], F32, "dx")
    within_norm(gw, ref["dw"], F32, "dw")
    flat = torch.full((4, 300), 7.25, device="cuda")
    assert not T.layer_norm(flat).any()                                   # no variance: 0, not NaN
    empty = torch.empty(0, 12, device="cuda", requires_grad=True)
    w = torch.ones(12, device="cuda", requires_grad=True)
    y = T.layer_norm(empty, w)
    g = torch.autograd.grad(y, (empty, w), torch.empty_like(y))
    assert y.shape == (0, 12) and g[0].shape == (0, 12) and not g[1].any()


def test_layer_norm_far_from_zero():
    """A mean of a thousand deviations: the variance is that of the deviations, not a difference of squares."""
    x = rnd(64, 512, seed=1) + 1000.0
    y = T.layer_norm(x)
    x64 = x.double()
    d = x64 - x64.mean(-1, keepdim=True)
    ref = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    assert (y.double() - ref).abs().max() <= 1000.0 * 2.0 ** -20     # the mean's own rounding, sixteen steps of 1000


# ---- rotary positions -------------------------------------------------------------------------------------------------------------
def rotary_64(x, positions, sections, interleaved, inverse=False):
    x = x.detach().cpu().double()
    y, terms, first = x.clone(), torch.zeros_like(x), 0
    for a, n in enumerate(sections):
        freq = 10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
        angle = (positions.cpu().double()[..., a, None] * freq)[..., None, :] * (-1 if inverse else 1)
        at = torch.arange(n // 2)
        lo, hi = (first + 2 * at, first + 2 * at + 1) if interleaved else (first + at, first + n // 2 + at)
        u, w = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = u * angle.cos() - w * angle.sin(), u * angle.sin() + w * angle.cos()
        terms[..., lo] = terms[..., hi] = u.abs() + w.abs()
        first += n
    return y, terms


def within_rotary(got, pair, dtype, what):
    """Three fp32 roundings of products and sum and two of sine and cosine, each of the pair's magnitude, then the stored one."""
    got, (ref, terms) = got.detach().double().cpu(), pair
    bound = STORED[dtype] * ref.abs() + 8 * 2.0 ** -24 * terms
    assert ((got - ref).abs() <= bound).all(), f"{what}: {float(((got - ref).abs() - bound).max()):.3e} over"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("D,sections", [(16, (8, 8)), (128, (32, 48, 48)), (64, (64,)), (80, (20, 30, 30)), (128, (16, 16)), (7, (2, 4)), (24, (2, 6, 4, 10)), (66, (6, 60))],
                         ids=lambda v: "_".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_rotary(D, sections, interleaved, dtype):
    B, L, H, Hk, n = 3, 37, 4, 2, len(sections)
    freqs = T.rotary_frequencies(sections)
    g = torch.Generator().manual_seed(D)
    for layout, kind, far in (("tokens", torch.int64, 50), ("heads", torch.int32, 2000000), ("odd", torch.float32, 300), ("packed", torch.int64, 10 ** 6)):
        q, k, _ = heads(layout, B, L, L, H, Hk, D, dtype, 1)
        shape = (L, n) if kind == torch.int32 else (B, L, n)
        positions = torch.randint(-far, far, shape, generator=g).to(kind)
        if kind == torch.float32:
            positions += 0.37
        positions = positions.cuda()
        dq, dk = rnd(B, L, H, D, seed=3, dtype=dtype), rnd(B, Hk, L, D, seed=4, dtype=dtype).transpose(1, 2)
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        qo, ko = T.rotary(q, k, positions, freqs, sections, interleaved)
        gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
        for name, got, x, inv in (("q", qo, q, False), ("k", ko, k, False), ("dq", gq, dq, True), ("dk", gk, dk, True)):
            within_rotary(got, rotary_64(x, positions, sections, interleaved, inv), dtype, f"{layout} {name}")
        rest = sum(sections)
        assert torch.equal(qo[..., rest:], q[..., rest:]) and torch.equal(gk[..., rest:], dk[..., rest:])


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0), (0, 0)])
def test_rotary_of_no_heads(H, Hk):
    q, k = rnd(2, 5, H, 8), rnd(2, 5, Hk, 8, seed=1)
    freqs, positions = T.rotary_frequencies((8,)), torch.arange(5, device="cuda")[:, None]
    qo, ko = T.rotary(q, k, positions, freqs, (8,))
    for got, x in ((qo, q), (ko, k)):
        assert got.shape == x.shape and got.dtype == x.dtype
        within_rotary(got, rotary_64(x, positions, (8,), False), F32, "no heads")


@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (64, 1, 32), (1, 1500, 5), (2, 1024, 4)])
def test_rotary_sizes_one_tensor_and_one_gradient(B, L, H):
    sections, D = (16, 24, 24), 64
    freqs, positions = T.rotary_frequencies(sections), torch.randint(0, 5000, (B, L, 3), device="cuda")
    x = rnd(B, L, H, D, seed=1).requires_grad_()
    y = T.rotary(x, None, positions, freqs, sections)
    within_rotary(y, rotary_64(x, positions, sections, False), F32, "alone")
    back, none = T.rotate(y.detach(), None, positions, freqs, sections, inverse=True)
    assert none is None and (back - x).abs().max() <= 16 * 2.0 ** -24 * 2 * x.abs().max()
    k = rnd(B, L, 2, D, seed=2).requires_grad_()
    qo, ko = T.rotary(x, k, positions, freqs, sections)
    assert torch.equal(qo, y)
    (only,) = torch.autograd.grad(ko, k, torch.ones_like(ko))             # q's result is not used
    within_rotary(only, rotary_64(torch.ones_like(ko), positions, sections, False, True), F32, "dk alone")


# ---- together ---------------------------------------------------------------------------------------------------------------------
SECTIONS = (8, 8)


def layer(p, x, positions, freqs, mask):
    """Pre-norm layer over [B, 16 * 64] image tokens: norm, projection, rotary over height and width, attention, residual, norm."""
    B, L, C = x.shape
    h = T.layer_norm(x, p["w1"], p["b1"])
    qkv = (h @ p["wqkv"]).view(B, L, 8, 16)
    q, k = T.rotary(qkv[:, :, :4], qkv[:, :, 4:6], positions, freqs, SECTIONS)
    a = T.attention(q, k, qkv[:, :, 6:], key_padding_mask=mask).reshape(B, L, 64)
    y, s = T.layer_norm(a @ p["wo"], p["w2"], p["b2"], residual=x)
    return y, s


def layer_64(p, x, positions, mask):
    def norm(t, w, b):
        d = t - t.mean(-1, keepdim=True)
        return d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * w + b

    def turn(t):
        parts, first = [], 0
        for a, n in enumerate(SECTIONS):
            angle = positions[:, a, None].double().cpu() * 10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
            c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]
            u, w = t[..., first:first + n // 2], t[..., first + n // 2:first + n]
            parts += [u * c - w * s, u * s + w * c]
            first += n
        return torch.cat(parts, -1)

    B, L, C = x.shape
    qkv = (norm(x, p["w1"], p["b1"]) @ p["wqkv"]).view(B, L, 8, 16)
    q, k, v = turn(qkv[:, :, :4]).transpose(1, 2), turn(qkv[:, :, 4:6]).transpose(1, 2), qkv[:, :, 6:].transpose(1, 2)
    s = (q @ k.repeat_interleave(2, 1).transpose(2, 3) * 0.25).masked_fill(mask.cpu()[:, None, None], -math.inf)
    a = (torch.softmax(s, -1) @ v.repeat_interleave(2, 1)).transpose(1, 2).reshape(B, L, 64)
    s = a @ p["wo"] + x
    return norm(s, p["w2"], p["b2"]), s


def layer_case(L=1024, B=2, seed=0):
    p = {"w1": rnd(64, seed=1) * 0.2 + 1, "b1": rnd(64, seed=2), "wqkv": rnd(64, 128, seed=3, scale=0.2), "wo": rnd(64, 64, seed=4, scale=0.2),
         "w2": rnd(64, seed=5) * 0.2 + 1, "b2": rnd(64, seed=6)}
    x = rnd(B, L, 64, seed=7 + seed)
    at = torch.arange(L, device="cuda")
    mask = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    mask[1:, L - L // 5:] = True
    return p, x, torch.stack((at // 64, at % 64), -1), T.rotary_frequencies(SECTIONS), mask


def test_layer_over_image_tokens_forward_and_gradients():
    p, x, positions, freqs, mask = layer_case()
    dy, ds = rnd(*x.shape, seed=30), rnd(*x.shape, seed=31)
    leaves = [t.requires_grad_() for t in (x, *p.values())]
    y, s = layer(p, x, positions, freqs, mask)
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    p64 = {n: t.detach().cpu().double().requires_grad_() for n, t in p.items()}
    x64 = x.detach().cpu().double().requires_grad_()
    y64, s64 = layer_64(p64, x64, positions, mask)
    want = torch.autograd.grad((y64, s64), (x64, *p64.values()), (dy.cpu().double(), ds.cpu().double()))
    for name, a, b in zip(("y", "s", "x", *p), (y, s, *grads), (y64, s64, *want)):
        off = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 1e-5, (name, off)     # five fp32 operators in a row, each some 1e-6 (a random walk of its roundings)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_operators_captured_and_replayed(dtype):
    """Forward and backward of all three in one graph, replayed on new data between eager work, equal to the eager result each time; two graphs share
    no workspace."""
    B, L, H, D = 2, 300, 4, 16
    freqs, at = T.rotary_frequencies(SECTIONS), torch.arange(L, device="cuda")
    positions, mask = torch.stack((at // 20, at % 20), -1), key_mask("lengths", B, L)
    w, b = rnd(64, seed=1) + 1, rnd(64, seed=2)

    def program(x, r, d):
        y, s, stat = T.layer_norm_forward(x, w, b, residual=r)
        h = y.view(B, L, H, D)
        q, k = T.rotate(h, h, positions, freqs, SECTIONS)
        out, lse = T.attention_forward(q, k, h, mask)
        dq, dk, dv = T.attention_backward(d.view(B, L, H, D), q, k, h, out, lse, mask)
        dq, dk = T.rotate(dq, dk, positions, freqs, SECTIONS, inverse=True)
        single, _ = T.attention_forward(q[:, :1], k, h, mask, need_saved=False)
        ds, dw, db = T.layer_norm_backward((dq + dk + dv).view(B, L, 64), s, w, stat, d)
        return out, dq, dk, dv, single, s, ds, dw, db

    def data(seed):
        return [rnd(B, L, 64, seed=seed + i, dtype=dtype) for i in range(3)]

    graphs = []
    for n in range(2):
        held = data(40 + n)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            program(*held)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = program(*held)
        graphs.append((g, held, res))
    for round_ in range(3):
        fresh = [data(60 + 10 * round_ + 5 * n) for n in range(2)]
        for (g, held, _), new in zip(graphs, fresh):
            for a, c in zip(held, new):
                a.copy_(c)
        for g, _, _ in graphs:
            g.replay()
        eager = [program(*new) for new in fresh]
        torch.cuda.synchronize()
        for (_, _, res), want in zip(graphs, eager):
            assert all(torch.equal(a, c) for a, c in zip(res, want)), round_


def test_attention_reads_long_sequences_where_they_lie():
    """Head-major keys of 20000 tokens (a head stride of 2.5 million elements), and tokens so far apart that a copy is made: the same result."""
    q = rnd(1, 4, 1, 128, seed=1, dtype=BF16).transpose(1, 2)
    k, v = (rnd(1, 2, 20000, 128, seed=s, dtype=BF16).transpose(1, 2) for s in (2, 3))
    assert T._laid_out(k, 1).data_ptr() == k.data_ptr() and T._laid_out(q, 1, 2).data_ptr() == q.data_ptr()
    want, lse = T.attention_forward(q, k.contiguous(), v.contiguous())
    got = T.attention_forward(q, k, v)
    assert torch.equal(got[0], want) and torch.equal(got[1][0], lse[0])
    far = torch.empty(40 << 22, dtype=BF16, device="cuda").as_strided((1, 40, 2, 128), (40 << 22, 1 << 22, 128, 1))
    far.copy_(k[:, :40])
    assert T._laid_out(far, 1).data_ptr() != far.data_ptr()
    assert torch.equal(T.attention_forward(q, far, far)[0], T.attention_forward(q, k[:, :40], k[:, :40])[0])


def test_no_gradient_of_a_gradient():
    """Asked for, it is refused: the backward pass is no function that autograd could differentiate."""
    x = rnd(4, 16, seed=1).requires_grad_()
    with pytest.raises(NotImplementedError, match="gradient of the gradient"):
        torch.autograd.grad(T.layer_norm(x).sum(), x, create_graph=True)
    q = rnd(1, 4, 2, 16, seed=1).requires_grad_()
    with pytest.raises(NotImplementedError, match="gradient of the gradient"):
        torch.autograd.grad(T.attention(q, q, q).sum(), q, create_graph=True)
    with pytest.raises(NotImplementedError, match="gradient of the gradient"):
        torch.autograd.grad(T.rotary(q, None, torch.zeros(4, 1, dtype=torch.int64, device="cuda"), T.rotary_frequencies((16,)), (16,)).sum(), q, create_graph=True)


@pytest.mark.parametrize("what", ["q", "positions", "sections", "freqs", "mask", "residual", "weight", "lse"])
def test_python_refusals_on_the_gpu(what):
    """Raised before any launch."""
    q, at, f = rnd(2, 5, 4, 16, seed=1), torch.zeros(5, 2, dtype=torch.int64, device="cuda"), T.rotary_frequencies((8, 8))
    x, w = rnd(6, 12, seed=2), torch.ones(12, device="cuda")
    calls = {
        "q": [lambda: T.attention(q.half(), q.half(), q.half()), lambda: T.attention(q, q.bfloat16(), q), lambda: T.attention(q, q[:1], q[:1]),
              lambda: T.attention(q[:, :, :3], q[:, :, :2], q[:, :, :2]), lambda: T.attention(*[rnd(1, 2, 1, 136)] * 3), lambda: T.attention(q, q, q[:, :4]),
              lambda: T.attention(q[0], q[0], q[0]), lambda: T.attention(q, q.cpu(), q), lambda: T.rotary(q[0], None, at, f, (8, 8))],
        "positions": [lambda: T.rotary(q, q, at[:4], f, (8, 8)), lambda: T.rotary(q, q, at.double(), f, (8, 8)), lambda: T.rotary(q, q, at.cpu(), f, (8, 8)),
                      lambda: T.rotary(q, q, at.expand(3, 5, 2), f, (8, 8)), lambda: T.rotary(q, q, at[:, :1], f, (8, 8))],
        "sections": [lambda: T.rotary(q, q, at, f, (8, 7)), lambda: T.rotary(q, q, at, f, (8, 10)), lambda: T.rotary(q, q, at, f, ()), lambda: T.rotary(q, q, at, f, (16, 0))],
        "freqs": [lambda: T.rotary(q, q, at, f.float(), (8, 8)), lambda: T.rotary(q, q, at, f[:7], (8, 8)), lambda: T.rotary(q, q, at, f.cpu(), (8, 8))],
        "mask": [lambda: T.attention(q, q, q, key_padding_mask=torch.zeros(2, 4, dtype=torch.bool, device="cuda")), lambda: T.attention(q, q, q, key_padding_mask=torch.zeros(2, 5, device="cuda")),
                 lambda: T.attention(q, q, q, key_padding_mask=torch.zeros(2, 5, dtype=torch.bool))],
        "residual": [lambda: T.layer_norm(x, residual=x[:5]), lambda: T.layer_norm(x, residual=x.bfloat16()), lambda: T.layer_norm(x[:, :0])],
        "weight": [lambda: T.layer_norm(x, w[:11]), lambda: T.layer_norm(x, w.bfloat16()), lambda: T.layer_norm(x, w, w.cpu()), lambda: T.layer_norm(x.double())],
        "lse": [lambda: T.attention_backward(q, q, q, q, q, (torch.zeros(2, 4, 4, device="cuda"), None)), lambda: T.attention_backward(q[:, :4], q, q, q, q, (torch.zeros(2, 4, 5, device="cuda"), None)),
                lambda: T.attention_backward(q, q, q, q, q, (torch.zeros(2, 4, 5, device="cuda"), q)),
                lambda: T.layer_norm_backward(x, x, w, torch.zeros(5, 2, device="cuda"))],
    }
    for call in calls[what]:
        with pytest.raises((RuntimeError, NotImplementedError), match="tatt_amd"):
            call()


def test_attention_gradients_in_bf16_are_not_those_of_a_rounded_output():
    """Few keys: dO . O of the stored output alone would be off by its rounding, as much as all other roundings together.  A rounding to bf16 is
    uniform over half a step, 2^-8 of the power of two below the value: 2^-8 / sqrt(3) / 1.4 = 1.6e-3 of it in the root mean square (1.4: that of
    mantissas between 1 and 2).  dQ and dK carry two independent ones, of dS and of the stored result: 2.3e-3 in the norm; 2.6e-3 leaves a tenth."""
    q, k, v = heads("tokens", 16, 300, 12, 4, 4, 64, BF16, 12)
    do = rnd(16, 300, 4, 64, seed=9, dtype=BF16)
    ref = attention_64(q, k, v, do, None, False, 0.125)
    out, saved = T.attention_forward(q, k, v)
    for name, got in zip(("dq", "dk"), T.attention_backward(do, q, k, v, out, saved)):
        off = float((got.double().cpu() - ref[name][0]).norm() / ref[name][0].norm())
        assert off <= 2.6e-3, (name, off)
