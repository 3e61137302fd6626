"""Attention's kernels where large or many problems choose them: 64 rows a wave, the few-row forms of a full chip, and a join of more splits than a wave
has lanes.  The conditions are those of the launch plans (mha_fwd.hip, mha_bwd.hip, plan() in mha.h) and are asserted, so that a case does not leave
its kernel behind when a plan changes."""
import pytest
import torch

from tatt_amd.lib import lib
from tatt_amd.model import token_ops as T

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


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,causal", [((3, 70, 333, 4, 2, 64), False), ((3, 300, 300, 2, 2, 32), True), ((3, 1, 900, 8, 2, 128), False)], ids=str)
def test_masks_of_any_strides(shape, causal, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v = heads("tokens", *shape, dtype, 24)
    do, hidden = rnd(B, Lq, H, D, seed=9, dtype=dtype), key_mask("holes", B, Lk)
    spaced = torch.ones(B, 2 * Lk, dtype=torch.bool, device="cuda")
    spaced[:, ::2] = hidden
    for mask in (hidden.t().contiguous().t(), spaced[:, ::2], hidden[:1].expand(B, Lk), hidden[:, :1].expand(B, Lk)):
        assert not mask.is_contiguous()
        saved = T.attention_forward(q, k, v, mask, causal)
        want = T.attention_forward(q, k, v, mask.contiguous(), causal)
        assert torch.equal(saved[0], want[0]) and torch.equal(saved[1][0], want[1][0])
        for a, b in zip(T.attention_backward(do, q, k, v, *saved, mask, causal), T.attention_backward(do, q, k, v, *want, mask.contiguous(), causal)):
            assert torch.equal(a, b)
    check_attention(q, k, v, do, spaced[:, ::2], causal, D ** -0.5, "spaced")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 1, 700, 8, 2, 128), (2, 150, 150, 4, 2, 128), (1, 600, 600, 2, 2, 96), (32, 300, 40, 8, 8, 64)], ids=lambda s: "x".join(map(str, s)))
def test_wide_heads_captured_and_replayed(shape, dtype):
    """Kernels with more than 64 KB of LDS, which is asked for at their launch, and splits with their join, in a graph that is replayed on new data between eager work."""
    B, Lq, Lk, H, Hk, D = shape
    mask = key_mask("lengths", B, Lk)

    def program(q, k, v, do):
        out, saved = T.attention_forward(q, k, v, mask)
        return (out, saved[0], *T.attention_backward(do, q, k, v, out, saved, mask))

    def data(seed):
        return [*heads("tokens", *shape, dtype, seed), rnd(B, Lq, H, D, seed=seed + 5, dtype=dtype)]

    held, side, graph = data(50), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        program(*held)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = program(*held)
    for seed in (60, 70, 80):
        fresh = data(seed)
        for a, b in zip(held, fresh):
            a.copy_(b)
        graph.replay()
        want = program(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
