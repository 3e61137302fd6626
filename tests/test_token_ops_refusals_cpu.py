"""Calls that the token operators would answer wrongly and refuse instead, checked without a GPU: every refusal comes before any launch."""
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from tatt_amd import lib as tl
from tatt_amd.model import token_ops as T

CALLS = {  # operator -> (its call, shapes of its tensors)
    "layer_norm": (lambda x, residual, weight, bias: T.layer_norm(x, weight, bias, residual=residual), ((3, 8), (3, 8), (8,), (8,))),
    "rotary": (lambda q, k, positions, freqs: T.rotary(q, k, positions, freqs, (8,)), ((1, 3, 2, 8), (1, 3, 1, 8), (3, 1), (4,))),
    "attention": (T.attention, ((1, 3, 2, 8), (1, 5, 2, 8), (1, 5, 2, 8))),
}


@pytest.mark.parametrize("op,at", [(op, at) for op, (_, shapes) in CALLS.items() for at in range(len(shapes))])
def test_forward_mode_derivatives_are_refused(op, at):
    """The result of a dual tensor would carry no tangent: a derivative of zero."""
    call, shapes = CALLS[op]
    with forward_ad.dual_level():
        args = [torch.randn(*s) for s in shapes]
        args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(NotImplementedError, match=f"tatt_amd {op}: no forward-mode"):
            call(*args)
    with pytest.raises(RuntimeError, match="GPU only"):      # not refused for it any more
        call(*(torch.randn(*s) for s in shapes))


@pytest.mark.parametrize("queries_too", [False, True])
@pytest.mark.parametrize("op,what", [("rotary", "positions"), ("rotary", "freqs"), ("attention", "scale"), ("layer_norm", "eps")])
def test_values_without_a_gradient_are_refused_where_they_require_one(op, what, queries_too):
    """autograd would leave the gradient None, or the whole result without one."""
    call, shapes = CALLS[op]
    args = [torch.randn(*s) for s in shapes]
    args[0].requires_grad_(queries_too)
    value = torch.tensor(0.5, requires_grad=True)
    if op == "rotary":
        args[{"positions": 2, "freqs": 3}[what]].requires_grad_()
    elif op == "attention":
        call = lambda q, k, v: T.attention(q, k, v, scale=value)    # noqa: E731
    else:
        call = lambda x, *_: T.layer_norm(x, eps=value)    # noqa: E731
    with pytest.raises(NotImplementedError, match=f"tatt_amd {op}: .*{what}.*no gradient"):
        call(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):      # nothing is lost here
        call(*args)


REFUSED = [  # B, Lq, Lk, H, Hkv, D: rows past 2^30, products past 31 and 64 bits, heads, widths
    (1, 1 << 16, 1, 1 << 16, 1, 8), (1, 1 << 15, 40, 1 << 16, 1, 8), (1, (1 << 31) - 1, 5, 2, 1, 8), (1, 1, (1 << 31) - 1, 1, 1, 8), (1 << 22, 1 << 21, 1, 1 << 21, 1 << 21, 8),
    (1 << 22, 1, 1 << 21, 1 << 21, 1 << 21, 8), (1, 1, 1, 1 << 17, 1, 8), (1, 1, 1, 1, 1, 129), (1, 1, 1, 3, 2, 8), (0, 1, 1, 1, 1, 8), (1, -1, 1, 1, 1, 8)]


def test_attention_workspace_queries_of_what_is_refused():
    """0, from a process that lives on: row counts past 31 bits ended it with a division by zero."""
    ask = "from tatt_amd.lib import lib; c = lib().cdll\n" + "\n".join(
        f"print(c.tatt_mha_{way}_workspace{(*dims, dtype)}, flush=True)" for dims in REFUSED for way in ("fwd", "bwd") for dtype in (0, 1))
    child = subprocess.run([sys.executable, "-c", ask], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=300)
    assert child.returncode == 0, (child.returncode, len(child.stdout.split()))
    assert child.stdout.split() == ["0"] * 4 * len(REFUSED)
    assert tl.lib().mha_bwd_workspace(2, 3, 5, 4, 2, 16, 0) >= 2 * 3 * 4       # what is taken has one


@pytest.mark.parametrize("dims", [d for d in REFUSED if min(d) > 0], ids=lambda d: "x".join(map(str, d)))
def test_attention_entry_points_refuse_the_same(dims):
    B, Lq, Lk, H, Hkv, D = dims
    p = 4096     # a stand-in for a device pointer: refused before it is used
    strides = (tl.ctypes.c_long * 15)()
    with pytest.raises(RuntimeError, match="tatt_mha_fwd: "):
        tl.lib().mha_fwd(p, p, p, strides, None, None, p, None, None, B, Lq, Lk, H, Hkv, D, 1.0, 0, 0, p, None)
    with pytest.raises(RuntimeError, match="tatt_mha_bwd: "):
        tl.lib().mha_bwd(p, p, p, strides, None, None, p, None, p, p, p, p, p, B, Lq, Lk, H, Hkv, D, 1.0, 0, 0, p, None)


FAR = (1 << 32) + 1     # its low 32 bits: 1


def meta(*shape):
    return torch.empty(1, dtype=torch.bfloat16, device="meta").expand(shape)


@pytest.mark.parametrize("op,call", [
    ("layer_norm", lambda: T.layer_norm(meta(1, FAR + 7))), ("layer_norm", lambda: T.layer_norm_backward(meta(1, FAR + 7), meta(1, FAR + 7), None, torch.empty(1, 2, device="meta"))),
    ("rotary", lambda: T.rotate(meta(FAR, 1, 1, 2), None, torch.empty(1, 1, device="meta"), torch.empty(1, dtype=torch.float64, device="meta"), (2,))),
    ("rotary", lambda: T.rotate(meta(1, 1, 1, 2), meta(1, 1, FAR, 2), torch.empty(1, 1, device="meta"), torch.empty(1, dtype=torch.float64, device="meta"), (2,))),
    ("rotary", lambda: T.rotate(meta(1, 1, 1, FAR), None, torch.empty(1, 1, device="meta"), torch.empty(1, dtype=torch.float64, device="meta"), (2,))),
    ("attention", lambda: T.attention_forward(meta(FAR, 1, 1, 8), meta(FAR, 1, 1, 8), meta(FAR, 1, 1, 8))),
    ("attention", lambda: T.attention_forward(meta(1, 1, 1, 8), meta(1, FAR, 1, 8), meta(1, FAR, 1, 8))),
    ("attention", lambda: T.attention_forward(meta(1, FAR, 1, 8), meta(1, 1, 1, 8), meta(1, 1, 1, 8))),
    ("attention", lambda: T.attention_forward(meta(1, 1, FAR, 8), meta(1, 1, 1, 8), meta(1, 1, 1, 8)))])
def test_dimensions_past_31_bits_are_refused(op, call, monkeypatch):
    """The C ABI's int would take the low 32 bits, and the call would leave all but the first rows unwritten.  Tensors without memory, and a stand-in for the
    launch: a call that gets that far is not refused."""
    monkeypatch.setattr(T, "_check", lambda what, t0, *tensors: 1)
    monkeypatch.setattr(T, "_call", lambda name, device, *args: pytest.fail(f"{name} would be launched"))
    with pytest.raises(RuntimeError, match=f"tatt_amd {op}: a dimension of 2.31"):
        call()


@pytest.mark.parametrize("C", [1 << 27, (1 << 31) - 1])
def test_layernorm_refuses_rows_past_its_loops(C):
    p = 4096     # a stand-in for a device pointer: refused before it is used
    with pytest.raises(RuntimeError, match="2.27 elements"):
        tl.lib().layernorm_fwd(p, C, None, 0, None, None, None, p, None, 1, C, 1e-5, 0, None)
    with pytest.raises(RuntimeError, match="2.27 elements"):
        tl.lib().layernorm_bwd(p, C, p, C, None, 0, None, p, p, None, None, 1, C, 0, None, None)
    assert tl.lib().layernorm_workspace(1, C, 0) == 0
