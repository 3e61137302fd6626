"""Calls that the token operators would answer wrongly and refuse instead, checked without a GPU: every refusal comes before any launch."""
import pytest
import torch
from torch.autograd import forward_ad

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
