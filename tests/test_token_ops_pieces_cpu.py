"""The three bf16 pieces that stand for an fp32 operand of attention's products, emulated: their six products are no further from 64 bits than a plain
fp32 computation, and without any one of them several times as far.  (test_gpu_token_ops_exact.py holds the kernels to that.)"""
import pytest
import torch

SIX = [(0, 2), (1, 1), (2, 0), (0, 1), (1, 0), (0, 0)]     # smallest first


def pieces(x):
    out = []
    for _ in range(3):
        out.append(x.bfloat16().float())
        x = x - out[-1]
    return out


def product(a, b, terms):
    """a b as the sum of piece products in fp32."""
    a, b, r = pieces(a), pieces(b), 0.0
    for i, j in terms:
        r = r + a[i] @ b[j]
    return r


def off(q, k, v, times):
    """softmax(q k^T) v with `times` for its products: the error against 64 bits in the norm."""
    k = k.transpose(-1, -2).contiguous()
    got = times(torch.softmax(times(q, k).double(), -1).float(), v).double()
    want = torch.softmax(q.double() @ k.double(), -1) @ v.double()
    return float((got - want).norm() / want.norm())


def test_three_pieces_hold_every_bit():
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.arange(4096) % 60 - 30.0)
    assert torch.equal(sum(p.double() for p in pieces(x)), x.double())


@pytest.mark.parametrize("scale", [None, 0.3])
@pytest.mark.parametrize("shape", [(26, 26, 16), (64, 40, 64), (100, 300, 128), (33, 1000, 96)], ids=str)
def test_six_products_and_not_five(shape, scale):
    Lq, Lk, D = shape
    g = torch.Generator().manual_seed(Lk)
    q, k, v = (torch.randn(4, n, D, generator=g) for n in (Lq, Lk, Lk))
    q = q * (D ** -0.5 if scale is None else scale)
    plain = off(q, k, v, torch.matmul)
    assert off(q, k, v, lambda a, b: product(a, b, SIX)) <= plain
    for gone in SIX:
        assert off(q, k, v, lambda a, b: product(a, b, [t for t in SIX if t != gone])) > 2.5 * plain, gone
