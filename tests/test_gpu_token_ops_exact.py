"""How exact the token operators are, in closer bounds than those of test_gpu_token_ops.py, which allow for every operand of a product in the
tensors' type."""
import math

import pytest
import torch

from tatt_amd.model import token_ops as T

from .test_gpu_token_ops import BF16, F32, STORED, attention_64, heads, key_mask, rnd

pytestmark = pytest.mark.gpu


def attention_in_bounds(q, k, v, do, mask, causal, scale, of_a_term):
    """out, dq, dk and dv are within STORED of the value (their own rounding) and `of_a_term` of the sum of the terms' magnitudes; the gradients take P
    from the stored fp32 lse, which is off by 2^-24 of itself, and P by as much as that."""
    ref = attention_64(q, k, v, do, mask, causal, scale)
    out, saved = T.attention_forward(q, k, v, mask, causal, scale)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *T.attention_backward(do, q, k, v, out, saved, mask, causal, scale))))
    seen = torch.isfinite(ref["lse"])
    of_lse = 2.0 ** -24 * float(ref["lse"][seen].abs().max()) if seen.any() else 0.0
    for name, g in got.items():
        value, terms = ref[name]
        bound = STORED[q.dtype] * value.abs() + (of_a_term + (0.0 if name == "out" else of_lse)) * terms + 1e-30
        off = (g.double().cpu() - value).abs() / bound
        assert off.max() <= 1, (name, float(off.max()))


@pytest.mark.parametrize("kind,causal", [("none", False), ("holes", True)], ids=["plain", "masked"])
@pytest.mark.parametrize("shape", [(2, 40, 26, 4, 4, 16), (2, 65, 33, 2, 1, 32), (2, 100, 70, 4, 2, 64), (1, 130, 257, 6, 2, 96), (2, 90, 200, 2, 2, 128), (2, 1, 700, 8, 2, 128),
                                   (32, 300, 40, 8, 8, 64), (1, 600, 600, 2, 2, 64)], ids=lambda s: "x".join(map(str, s)))
def test_attention_in_bf16_rounds_only_what_it_stores(shape, kind, causal):
    """The probabilities and the gradient of the scores are computed values that no caller gave in bf16.  As two bf16 pieces they are off by
    2^-8 x 2^-8 = 2^-16 of themselves, with 2^-15 for the fp32 sums (a score of 128 products: 2e-6); as one piece by 2^-8, 85 times the bound."""
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", *shape, BF16, 21)
    attention_in_bounds(q, k, v, rnd(B, Lq, H, D, seed=9, dtype=BF16), key_mask(kind, B, Lk), causal, D ** -0.5, 2.0 ** -16 + 2.0 ** -15)


def plain_fp32(q, k, v, do, scale):
    """out, dq, dk and dv by torch's fp32 products."""
    q, k, v, do = (t.transpose(1, 2).contiguous() for t in (q, k, v, do))
    p = torch.softmax(q @ k.transpose(2, 3).contiguous() * scale, -1)
    out = p @ v
    ds = p * (do @ v.transpose(2, 3).contiguous() - (do * out).sum(-1, keepdim=True)) * scale
    return [t.transpose(1, 2) for t in (out, ds @ k, ds.transpose(2, 3).contiguous() @ q, p.transpose(2, 3).contiguous() @ do)]


@pytest.mark.parametrize("scale", [None, 0.3])
@pytest.mark.parametrize("shape", [(4, 26, 26, 4, 4, 16), (4, 64, 40, 4, 4, 64), (2, 100, 300, 4, 4, 128), (2, 33, 1000, 2, 2, 96), (1, 1024, 1024, 4, 4, 64), (2, 300, 20, 2, 2, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_attention_in_fp32_is_as_exact_as_plain_fp32(shape, scale):
    """In the norm.  Emulated, the six products of three pieces are at 0.4 to 0.6 of the plain form's error and any five of them at three times it or more
    (test_token_ops_pieces_cpu.py): 1.25 is between.  The gradients take P from the stored lse, base 2 and rounded to fp32: uniform over half a step, 2^-24 of the
    power of two above it / sqrt(3), which is ln 2 times that of a row's P and, the rows' roundings being independent, of a gradient (1000 keys: 1.9e-7)."""
    B, Lq, Lk, H, Hk, D = shape
    scale = D ** -0.5 if scale is None else scale
    q, k, v = heads("tokens", *shape, F32, 22)
    do = rnd(B, Lq, H, D, seed=9)
    ref = attention_64(q, k, v, do, None, False, scale)
    out, saved = T.attention_forward(q, k, v, scale=scale)
    own = (out, *T.attention_backward(do, q, k, v, out, saved, scale=scale))
    of_lse = 2.0 ** (math.ceil(math.log2(float(ref["lse"].abs().max()) / math.log(2.0))) - 24) * math.log(2.0) / math.sqrt(3.0)
    for name, a, b in zip(("out", "dq", "dk", "dv"), own, plain_fp32(q, k, v, do, scale)):
        value = ref[name][0]
        a, b = (float((t.double().cpu() - value).norm() / value.norm()) for t in (a, b))
        assert a <= 1.25 * b + (0.0 if name == "out" else of_lse), (name, a, b, of_lse)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_layer_norm_of_rows_past_the_grid(dtype):
    """More columns than 65535 workgroups of 256 take at once.  Values of 1 and -1 in turn: mean 0 and variance 1 without rounding, and every result one product
    of 1 / sqrt(1 + eps), which fp32 holds to a few roundings."""
    R, C = 3, 65535 * 256 + 4098
    x = torch.ones(R, C, dtype=dtype, device="cuda")
    x[:, ::2] = -1
    dy = (torch.arange(R * C, device="cuda") % 7 - 3).view(R, C).to(dtype)
    y, s, stat = T.layer_norm_forward(x)
    dx, dw, db = T.layer_norm_backward(dy, s, None, stat)
    r = (1 + 1e-5) ** -0.5
    assert (y.float() - x.float() * r).abs().max() <= STORED[dtype] + 2.0 ** -21
    g = dy.double()
    assert (dw.double() - (g * x.double()).sum(0) * r).abs().max() <= 9 * 2.0 ** -21 and torch.equal(db.double(), g.sum(0))
    want = r * (g - g.mean(1, keepdim=True) - x.double() * r * (g * x.double() * r).mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= STORED[dtype] * want.abs() + 2.0 ** -18).all()


@pytest.mark.parametrize("C,n", [(64, 4), (200, 16)])
def test_layer_norm_parameter_sums(C, n):
    """65536 rows, n to a thread.  A rounding is uniform over half a step: e = 2^-24 / sqrt(3) / 1.4 = 2.5e-8 of its value in the root mean square.  Relative to the
    sum of all terms: xhat's two roundings e each and rstd's, uniform over a whole step as rsqrt's may be, 2 e, with half of its argument's: 2.5 e.  A thread's k-th
    addition is off by e of a sum of k random terms, sqrt(k) of one: sqrt(sum of k / n) = sqrt((n + 1) / 2) e, 1.6 e and 2.9 e.  A workgroup's partial sum and the result
    e each: 3.3 e and 4.1 e.  The sizes of partial sums are those of a random walk, whose spread moves that by up to a quarter."""
    x, w, dy = rnd(65536, C, seed=31, scale=1.5), rnd(C, seed=32) * 0.2 + 1, rnd(65536, C, seed=33)
    _, s, stat = T.layer_norm_forward(x, w, None)
    _, dw, db = T.layer_norm_backward(dy, s, w, stat)
    x64, g = x.double(), dy.double()
    var, mean = torch.var_mean(x64, dim=1, correction=0, keepdim=True)
    most = 1.25 * 2.5e-8 * (2.5 ** 2 + (n + 1) / 2 + 2) ** 0.5
    for got, ref in ((dw, (g * (x64 - mean) / torch.sqrt(var + 1e-5)).sum(0)), (db, g.sum(0))):
        off = float((got.double() - ref).norm() / ref.norm())
        assert off <= most, off


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("C", [8, 64, 200, 1024, 4096, 20001])
def test_layer_norm_bias_gradient_of_whole_numbers(C, dtype):
    """Whole numbers below 2^18, at most 64 rows of them to a workgroup: its sums stay below 2^24 and need no rounding, and the sum of all, 2^31 or so, is
    rounded once.  (Summed in fp32 the workgroups' sums would be rounded again and again.)"""
    R, g = 16384 if C > 1024 else 65536, torch.Generator(device="cuda").manual_seed(C)
    dy = (torch.randint(0, 256, (R, C), generator=g, device="cuda") << torch.randint(0, 11, (R, C), generator=g, device="cuda")).to(dtype)
    s = torch.ones(1, C, dtype=dtype, device="cuda").expand(R, C)
    _, _, db = T.layer_norm_backward(dy, s, None, torch.zeros(R, 2, device="cuda"))
    assert torch.equal(db, dy.double().sum(0).float())
