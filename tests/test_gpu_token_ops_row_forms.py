"""Every form of layer norm's and rotary's kernels: threads and chunks of a row, 16-byte accesses or single elements, with and without the parameters' gradients;
units of 16 and 8 bytes, and heads with more pairs than a workgroup's LDS holds turns for."""
import pytest
import torch

from tatt_amd.lib import lib
from tatt_amd.model import token_ops as T

from .test_gpu_token_ops import BF16, F32, norm_64, rnd, rotary_64, within_norm, within_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("short", [0, 1, 3], ids=["whole", "less1", "less3"])
@pytest.mark.parametrize("chunks", [1, 8, 9, 13, 32, 33, 50, 64, 65, 100, 128, 129, 200, 400, 512, 513, 900, 1025, 2048, 2049])
def test_layer_norm_forms(chunks, short, dtype):
    """Widths of `chunks` 16-byte pieces, and of a few elements less: 8 to 1024 threads of a row, one or two chunks each, and past 2048 none."""
    C, R = chunks * (8 if dtype == BF16 else 4) - short, 37 if chunks > 300 else 533
    x, r, dy, ds = (rnd(R, C, seed=40 + i, dtype=dtype) for i in range(4))
    w, b = rnd(C, seed=44) * 0.3 + 1, rnd(C, seed=45)
    for residual in (None, r):
        y, s, stat = T.layer_norm_forward(x, w, b, residual=residual)
        add = None if residual is None else ds
        dx, dw, db = T.layer_norm_backward(dy, s, w, stat, add)
        alone, none, _ = T.layer_norm_backward(dy, s, w, stat, add, need_params=False)
        assert none is None and torch.equal(alone, dx)
        ref = norm_64(s, w, b, dy, add, 1e-5)
        for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
            within_norm(got, ref[name], dtype if name in ("y", "dx") else F32, name)


@pytest.mark.parametrize("C", [64, 100, 9000])
def test_layer_norm_one_parameter_gradient(C):
    """The C ABI writes either alone, and leaves the other where it is."""
    x, dy = rnd(300, C, seed=1), rnd(300, C, seed=2)
    _, s, stat = T.layer_norm_forward(x)
    dx, dw, db = T.layer_norm_backward(dy, s, None, stat)
    work = torch.empty(lib().layernorm_workspace(300, C, 0), device="cuda")
    for a, b in ((torch.empty_like(dw), None), (None, torch.empty_like(db))):
        got = torch.empty_like(dx)
        lib().layernorm_bwd(s, C, dy, C, None, 0, None, stat, got, a, b, 300, C, 0, work)
        assert torch.equal(got, dx) and (a is None or torch.equal(a, dw)) and (b is None or torch.equal(b, db))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("D,sections", [(16, (16,)), (12, (12,)), (20, (4, 12)), (24, (8, 8)), (14, (6, 8)), (8, (2, 2, 4)), (1280, (1100,)), (1264, (600, 660)), (2048, (2048,)),
                                        (1050, (1042,)), (1101, (40, 1050))], ids=lambda v: "_".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_rotary_forms(D, sections, interleaved, dtype):
    B, L, H, Hk = 2, 21, 3, 1
    freqs, positions = T.rotary_frequencies(sections), torch.randint(-4000, 4000, (B, L, len(sections)), generator=torch.Generator().manual_seed(D)).cuda()
    q, k = rnd(B, L, H, D, seed=1, dtype=dtype), rnd(B, L, Hk, D, seed=2, dtype=dtype)
    for inverse in (False, True):
        qo, ko = T.rotate(q, k, positions, freqs, sections, interleaved, inverse)
        within_rotary(qo, rotary_64(q, positions, sections, interleaved, inverse), dtype, "q")
        within_rotary(ko, rotary_64(k, positions, sections, interleaved, inverse), dtype, "k")
