"""How exact the token operators are, in closer bounds than those of test_gpu_token_ops.py, which allow for every operand of a product in the
tensors' type."""
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
