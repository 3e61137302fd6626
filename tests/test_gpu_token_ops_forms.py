"""Attention's kernels where large or many problems choose them: 64 rows a wave, the few-row forms of a full chip, and a join of more splits than a wave
has lanes.  The conditions are those of the launch plans (mha_fwd.hip, mha_bwd.hip, plan() in mha.h) and are asserted, so that a case does not leave
its kernel behind when a plan changes."""
import pytest

from tatt_amd.lib import lib

from .test_gpu_token_ops import BF16, F32, check_attention, heads, key_mask, rnd
from .test_gpu_token_ops_exact import attention_in_bounds

pytestmark = pytest.mark.gpu


def splits(B, Lq, Lk, H, Hk, D, dtype):
    """of the forward pass, from its workspace: split by split the sums of D values, the maximum and the sum of every row"""
    return max(1, lib().mha_fwd_workspace(B, Lq, Lk, H, Hk, D, int(dtype == BF16)) // (B * H * Lq * (D + 2)))


def both_bounds(shape, dtype, kind, causal):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", *shape, dtype, 23)
    do, mask, scale = rnd(B, Lq, H, D, seed=9, dtype=dtype), key_mask(kind, B, Lk), D ** -0.5
    check_attention(q, k, v, do, mask, causal, scale, kind)
    if dtype == BF16:
        attention_in_bounds(q, k, v, do, mask, causal, scale, 2.0 ** -16 + 2.0 ** -15)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("kind", ["none", "lengths", "holes"])
@pytest.mark.parametrize("shape", [(32, 300, 77, 8, 8, 16), (32, 300, 90, 8, 8, 32), (32, 300, 300, 8, 8, 64), (16, 257, 140, 32, 16, 40), (44, 101, 130, 9, 3, 64), (64, 290, 33, 5, 5, 64),
                                   (26, 70, 65, 40, 5, 16)], ids=lambda s: "x".join(map(str, s)))
def test_64_rows_a_wave(shape, kind, causal):
    """bf16 heads up to 64 with a workgroup of 256 rows for every CU, forward and dQ: last blocks of 1 to 48 rows, groups of 1, 2, 3 and 8 heads, a padded width."""
    B, Lq, _, H, Hk, D = shape
    assert D <= 64 and B * Hk * -(-(Lq * (H // Hk)) // 256) >= 256      # more with splits
    both_bounds(shape, BF16, kind, causal)


@pytest.mark.parametrize("kind", ["none", "lengths", "holes"])
@pytest.mark.parametrize("D,causal", [(64, False), (64, True), (96, False), (128, True), (128, False)])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk", [(64, 1, 150, 8, 8), (48, 2, 333, 88, 11)], ids=lambda v: str(v))
def test_few_rows_in_fp32_on_a_full_chip(B, Lq, Lk, H, Hk, D, kind, causal):
    """One wave (heads past 64) or two along the keys where 512 workgroups or more fill the chip."""
    assert Lq * (H // Hk) <= 32 and B * Hk * splits(B, Lq, Lk, H, Hk, D, F32) >= 512
    both_bounds((B, Lq, Lk, H, Hk, D), F32, kind, causal)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "lengths", "most"])
@pytest.mark.parametrize("shape", [(2, 3, 200, 4, 2, 96), (2, 300, 20, 2, 2, 96), (1, 40, 31, 2, 1, 96), (2, 300, 32, 2, 2, 128)], ids=lambda s: "x".join(map(str, s)))
def test_few_rows_or_keys_of_heads_of_96_and_128(shape, kind, dtype):
    B, Lq, Lk, H, Hk, D = shape
    assert B * Hk * splits(*shape, dtype) < 512
    both_bounds(shape, dtype, kind, False)


@pytest.mark.parametrize("kind", ["none", "lengths", "holes"])
@pytest.mark.parametrize("shape,dtype", [((1, 1, 20000, 1, 1, 64), F32), ((1, 1, 20001, 2, 1, 128), F32), ((2, 1, 17000, 1, 1, 16), F32), ((1, 1, 70000, 1, 1, 16), BF16), ((1, 3, 70000, 2, 1, 24), BF16)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v)[-4:])
def test_more_splits_than_lanes(shape, dtype, kind):
    """The join takes the splits 64 at a time."""
    assert splits(*shape, dtype) > 64
    both_bounds(shape, dtype, kind, False)
