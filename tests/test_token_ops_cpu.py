"""What the token operators refuse, checked without a GPU: every refusal comes before any launch."""
import ctypes

import pytest
import torch

from tatt_amd import lib as tl
from tatt_amd.model import token_ops as T

L3, L9, L15 = (ctypes.c_long * n for n in (3, 9, 15))
P = 4096     # a stand-in for a device pointer: the calls below are refused before it is used


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 5, 2, 16)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.attention(x, x, x)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.layer_norm(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.rotary(x, x, torch.zeros(5, 1, dtype=torch.int64), T.rotary_frequencies((16,), device="cpu"), (16,))


def fwd(**kw):
    a = dict(q=P, k=P, v=P, strides=L9(), mask=None, mask_strides=None, out=P, low=None, lse=None, B=1, Lq=1, Lk=1, H=1, Hkv=1, D=16, scale=1.0, causal=0, dtype=0, ws=None)
    a.update(kw)
    tl.lib().mha_fwd(*a.values(), None)


def bwd(**kw):
    a = dict(q=P, k=P, v=P, strides=L15(), mask=None, mask_strides=None, out=P, low=None, dout=P, lse=P, dq=P, dk=P, dv=P, B=1, Lq=1, Lk=1, H=1, Hkv=1, D=16,
             scale=1.0, causal=0, dtype=0, ws=P)
    a.update(kw)
    tl.lib().mha_bwd(*a.values(), None)


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("kw,text", [({"q": None}, "bad arguments"), ({"v": None}, "bad arguments"), ({"strides": None}, "bad arguments"), ({"out": None}, "mha"),
                                     ({"B": 0}, "bad arguments"), ({"Lk": 0}, "bad arguments"), ({"Lq": -3}, "bad arguments"), ({"H": 3, "Hkv": 2}, "multiple"), ({"H": 1 << 17}, "65536"),
                                     ({"low": P}, "out_low"), ({"dtype": 1, "low": P + 2}, "out_low"), ({"D": 129}, "1 to 128"), ({"D": 0}, "1 to 128"), ({"dtype": 2}, "element type"), ({"mask": P}, "strides"),
                                     ({"B": 1 << 20, "Lq": 1 << 12}, "2\\^30"), ({"B": 1 << 20, "Lk": 1 << 12}, "2\\^30")])
def test_attention_entry_points_refuse(call, kw, text):
    with pytest.raises(RuntimeError, match=text):
        call(**kw)


@pytest.mark.parametrize("kw", [{"ws": None}, {"lse": None}, {"dq": None}, {"dout": None}])
def test_attention_backward_refuses_missing_buffers(kw):
    with pytest.raises(RuntimeError, match="tatt_mha_bwd"):
        bwd(**kw)


def test_layernorm_entry_points_refuse():
    L = tl.lib()
    ok = [P, 64, None, 0, None, None, None, P, None, 4, 64, 1e-5, 0]
    for at, bad, text in ((0, None, "bad arguments"), (7, None, "bad arguments"), (9, 0, "bad arguments"), (10, 0, "bad arguments"), (1, 63, "bad arguments"),
                          (2, P, "bad arguments"), (12, 5, "element type")):
        args = list(ok)
        args[at] = bad
        with pytest.raises(RuntimeError, match=text):
            L.layernorm_fwd(*args, None)
    ok = [P, 64, P, 64, None, 0, None, P, P, None, None, 4, 64, 0, None]
    for at, bad, text in ((0, None, "bad arguments"), (2, None, "bad arguments"), (7, None, "bad arguments"), (8, None, "bad arguments"), (3, 10, "bad arguments"),
                          (9, P, "workspace"), (13, 7, "element type"), (12, -1, "bad arguments")):
        args = list(ok)
        args[at] = bad
        with pytest.raises(RuntimeError, match=text):
            L.layernorm_bwd(*args, None)


def test_rotary_entry_point_refuses():
    L = tl.lib()

    def call(q=P, k=None, ks=None, ko=None, Hk=0, pos=P, pt=0, freqs=P, sections=(8, 8), naxes=None, B=1, Ln=4, D=16, dtype=0):
        s = (ctypes.c_int * max(1, len(sections)))(*sections)
        L.rotary(q, L3(), P, 2, k, ks, ko, Hk, pos, pt, L3(), freqs, s, len(sections) if naxes is None else naxes, B, Ln, D, 0, 0, dtype, None)

    for kw, text in (({"q": None}, "bad arguments"), ({"pos": None}, "bad arguments"), ({"freqs": None}, "bad arguments"), ({"k": P}, "k without"),
                     ({"pt": 3}, "position type"), ({"dtype": 9}, "element type"), ({"sections": (8, 7)}, "even"), ({"sections": (8, 0)}, "even"),
                     ({"sections": (8, 10)}, "exceed"), ({"naxes": 0}, "axes"), ({"sections": (2,) * 5}, "axes"), ({"B": 0}, "bad arguments"),
                     ({"B": 1 << 20, "Ln": 1 << 12}, "tokens")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)


def test_frequencies():
    f = T.rotary_frequencies((4, 8), base=100.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)


@pytest.mark.parametrize("call,n", [(fwd, 9), (bwd, 15)])
@pytest.mark.parametrize("kw", [{"D": 6}, {"q": P + 8}, {"k": P + 4}, {"strides": 2}, {"strides": 1 << 25}])
def test_attention_entry_points_refuse_rows_they_cannot_read(call, n, kw):
    if "strides" in kw:
        kw = {"strides": (ctypes.c_long * n)(*[kw["strides"]] * n)}
    with pytest.raises(RuntimeError, match="16-byte aligned places"):
        call(**kw)
