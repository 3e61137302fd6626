"""Operators of a transformer layer over image or text tokens, on the HIP kernels: `layer_norm` (any width, with the residual sum in
front), `rotary` (positions over several axes: height and width of a map, time of a clip) and `attention` (any lengths, head counts and
masks).  The interpreter's own layers (transformer_v2.py) run on kernels built for 64 channels, 4 heads x 16 and 26 keys; these are for layers
of any other size, in fp32 or bf16 (parameters, statistics and sums are fp32).

`layer_norm`, `rotary` and `attention` take part in autograd.  The pairs `*_forward` / `*_backward` are the same launches without it, as the
engine issues them: explicit outputs, capturable into a hipGraph.  (A `loss.backward()` inside a capture adds to leaves through nodes that an
earlier eager graph of the same leaves may still hold on another stream; take gradients there with the pairs, or with
torch.autograd.grad on leaves of the captured program's own.)  Everything runs on the current stream of the tensors' device; results are
bit-reproducible."""
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from ..lib import current_stream, lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_POS_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2}
_L2, _L3, _L9, _L15 = (ctypes.c_long * n for n in (2, 3, 9, 15))
_sections = functools.lru_cache(maxsize=64)(lambda sections: (ctypes.c_int * len(sections))(*sections))   # as the C ABI reads them


def _check(what, t0, *tensors):
    """The tensors' common element type (as the C ABI's number); raises for what the kernels do not take."""
    dtype, device = t0.dtype, t0.device
    if device.type != "cuda":
        raise RuntimeError(f"tatt_amd {what} runs on the GPU only (no CPU fallback)")
    for t in tensors:
        if t is not None and (t.dtype != dtype or t.device != device):
            raise RuntimeError(f"tatt_amd {what}: tensors of one type on one device expected, got {dtype} on {device} and {t.dtype} on {t.device}")
    code = _DTYPES.get(dtype)
    if code is None:
        raise NotImplementedError(f"tatt_amd {what}: float32 or bfloat16 tensors, got {dtype}")
    return code


def _call(name, device, *args):
    """A C entry point, tensors given as pointers, on the current stream of `device`."""
    L, index = lib(), device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _call(name, device, *args)
    rc = getattr(L.cdll, name)(*args, current_stream(index))
    if rc:
        raise RuntimeError(f"{name} failed ({rc}): {L.cdll.tatt_last_error().decode()}")


def _first_order(what):
    if torch.is_grad_enabled():      # create_graph=True: the gradient would be taken for a constant
        raise NotImplementedError(f"tatt_amd {what}: no gradient of the gradient")


def _int(what, *sizes):
    if max(sizes) >> 31:
        raise RuntimeError(f"tatt_amd {what}: a dimension of 2^31 or more, got {sizes}")      # the C ABI would get its low 32 bits


def _no_tangent(what, *tensors):
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"tatt_amd {what}: no forward-mode derivatives")      # the result would have none, as if they were zero


def _constant(what, required):
    if required and torch.is_grad_enabled():
        raise NotImplementedError(f"tatt_amd {what}: no gradient of a value that requires one")     # autograd would leave it None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t):
    """t with a contiguous last dimension (a copy only if it has none)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ---- layer norm -------------------------------------------------------------------------------------------------------------------
def _matrix(t):
    """(t as rows, elements between rows): any leading dimensions that one stride covers, else a contiguous copy."""
    C = t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and (t.stride(0) >= C or t.stride(0) == 0):
        return t, t.stride(0)
    return t.contiguous(), C


def _parameters(what, x, weight, bias):
    for n, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != x.shape[-1:] or p.dtype != torch.float32 or p.device != x.device or not p.is_contiguous()):
            raise RuntimeError(f"tatt_amd {what}: {n} is a contiguous float32 vector of the last dimension on the input's device, got {tuple(p.shape)} {p.dtype} on {p.device}")


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None, need_stat=True):
    """-> (y, sum, stat): y = LayerNorm(sum) over the last dimension, sum = x + residual in x's type (x itself without a residual), stat
    [rows, 2] fp32 = (mean, 1/sqrt(var + eps)) for layer_norm_backward (None unless need_stat)."""
    dtype = _check("layer_norm", x, residual)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError("tatt_amd layer_norm: the last dimension is empty")
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"tatt_amd layer_norm: the residual has the shape of x, got {tuple(residual.shape)} and {tuple(x.shape)}")
    _parameters("layer_norm", x, weight, bias)
    C = x.shape[-1]
    _int("layer_norm", C)
    R = x.numel() // C
    y = _like(x)
    s = _like(x) if residual is not None else x
    stat = torch.empty((R, 2), dtype=torch.float32, device=x.device) if need_stat else None
    if R:
        xm, ldx = _matrix(x)
        rm, ldr = (None, 0) if residual is None else _matrix(residual)
        _call("tatt_layernorm_fwd", x.device, xm.data_ptr(), ldx, _ptr(rm), ldr, _ptr(weight), _ptr(bias), None if residual is None else s.data_ptr(),
              y.data_ptr(), _ptr(stat), R, C, eps, dtype)
    return y, s, stat


def layer_norm_backward(dy, s, weight, stat, dsum=None, need_params=True):
    """-> (ds, dweight, dbias) of layer_norm_forward: ds = the gradient of the sum (x's and the residual's alike), with dsum, what reaches the
    sum by other ways, added; dweight and dbias fp32 (None unless need_params)."""
    dtype = _check("layer_norm", s, dy, dsum)
    _parameters("layer_norm", s, weight, None)
    C = s.shape[-1]
    _int("layer_norm", C)
    R = s.numel() // C
    if dy.shape != s.shape or (dsum is not None and dsum.shape != s.shape) or stat.shape != (R, 2) or stat.dtype != torch.float32 or stat.device != s.device or not stat.is_contiguous():
        raise RuntimeError("tatt_amd layer_norm_backward: dy and dsum have the shape of the sum, stat is layer_norm_forward's")
    ds, dw, db = _like(s), None, None
    if need_params:
        new = torch.empty if R else torch.zeros
        dw, db = (new(C, dtype=torch.float32, device=s.device) for _ in range(2))
    if R:
        sm, lds = _matrix(s)
        dym, lddy = _matrix(dy)
        dm, ldd = (None, 0) if dsum is None else _matrix(dsum)
        ws = torch.empty(lib().cdll.tatt_layernorm_workspace(R, C, dtype), dtype=torch.float32, device=s.device) if need_params else None
        _call("tatt_layernorm_bwd", s.device, sm.data_ptr(), lds, dym.data_ptr(), lddy, _ptr(dm), ldd, _ptr(weight), stat.data_ptr(), ds.data_ptr(),
              _ptr(dw), _ptr(db), R, C, dtype, _ptr(ws))
    return ds, dw, db


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        y, s, stat = layer_norm_forward(x, weight, bias, eps, residual)
        ctx.save_for_backward(s, weight, stat)
        return y if residual is None else (y, s)

    @staticmethod
    def backward(ctx, dy, dsum=None):
        _first_order("layer_norm")
        s, weight, stat = ctx.saved_tensors
        _, need_r, need_w, need_b, _ = ctx.needs_input_grad
        if dy is None:                                     # only the sum was used
            return dsum, dsum if need_r else None, None, None, None
        ds, dw, db = layer_norm_backward(dy, s, weight, stat, dsum, need_w or need_b)
        return ds, ds if need_r else None, dw if need_w else None, db if need_b else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """LayerNorm over the last dimension of x (float32 or bfloat16; weight and bias float32 or None), of any width below 2^27.  With a residual:
    -> (LayerNorm(sum), sum), sum = x + residual rounded to x's type, in one pass."""
    _no_tangent("layer_norm", x, residual, weight, bias, eps)
    _constant("layer_norm: eps", isinstance(eps, torch.Tensor) and eps.requires_grad)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        return _LayerNormFn.apply(x, residual, weight, bias, eps)
    y, s, _ = layer_norm_forward(x, weight, bias, eps, residual, need_stat=False)
    return y if residual is None else (y, s)


# ---- rotary positions -------------------------------------------------------------------------------------------------------------
def rotary_frequencies(sections, base=10000.0, device="cuda"):
    """Radians per position of every pair, float64 [sum(sections) / 2]: base ** (-2 i / section) for pair i of its section."""
    return torch.cat([base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n in sections]).to(device)


def rotate(q, k, positions, freqs, sections, interleaved=False, inverse=False):
    """`rotary` without autograd; inverse=True turns back (its backward pass)."""
    dtype = _check("rotary", q, k)
    n, width = len(sections), sum(sections)
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise RuntimeError("tatt_amd rotary: q [B, L, H, D] and k [B, L, Hk, D] expected")
    B, L, H, D = q.shape
    _int("rotary", B, H, D, 0 if k is None else k.shape[2])
    if not 1 <= n <= 4 or min(sections) <= 0 or any(s & 1 for s in sections) or width > D:
        raise RuntimeError(f"tatt_amd rotary: one to four positive even sections of at most {D} dimensions together, got {tuple(sections)}")
    kind, shape, device = _POS_TYPES.get(positions.dtype), positions.shape, q.device
    if kind is None:
        raise NotImplementedError(f"tatt_amd rotary: positions are int64, int32 or float32, got {positions.dtype}")
    if positions.device != device or shape[-2:] != (L, n) or len(shape) not in (2, 3) or (len(shape) == 3 and shape[0] not in (1, B)):
        raise RuntimeError(f"tatt_amd rotary: positions [L, axes] or [B, L, axes] on the tensors' device expected, got {tuple(shape)} on {positions.device}")
    if freqs.dtype != torch.float64 or freqs.shape != (width // 2,) or freqs.device != device or not freqs.is_contiguous():
        raise RuntimeError("tatt_amd rotary: freqs is a contiguous float64 vector of sum(sections) / 2 on the tensors' device (rotary_frequencies)")
    if H == 0 and k is not None:
        return _like(q), rotate(k, None, positions, freqs, sections, interleaved, inverse)[0]
    qo, ko = _like(q), None if k is None else _like(k)
    if qo.numel():
        q, k = _rows(q), None if k is None or not ko.numel() else _rows(k)
        sp = positions.stride()
        pos_strides = _L3(sp[0] if len(sp) == 3 and shape[0] > 1 else 0, sp[-2], sp[-1])
        _call("tatt_rotary", device, q.data_ptr(), _L3(*q.stride()[:3]), qo.data_ptr(), H, _ptr(k), None if k is None else _L3(*k.stride()[:3]), _ptr(ko),
              0 if k is None else k.shape[2], positions.data_ptr(), kind, pos_strides, freqs.data_ptr(), _sections(tuple(sections)), n, B, L, D,
              bool(interleaved), bool(inverse), dtype)
    return qo, ko


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, sections, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        ctx.how = (sections, interleaved)
        qo, ko = rotate(q, k, positions, freqs, sections, interleaved)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, dq, dk=None):
        _first_order("rotary")
        positions, freqs = ctx.saved_tensors
        if dq is None and dk is None:
            return (None,) * 6
        a, b = (dq, dk) if dq is not None else (dk, None)
        a, b = rotate(a, b, positions, freqs, *ctx.how, inverse=True)
        return (a, b, None, None, None, None) if dq is not None else (None, a, None, None, None, None)


def rotary(q, k, positions, freqs, sections, interleaved=False):
    """Rotary positions over several axes.  q [B, L, H, D] and k [B, L, Hk, D] or None (float32 or bfloat16, any strides); positions
    [L, axes] or [B, L, axes], int64, int32 or float32; the first sections[0] dimensions of each head turn by positions[..., 0], the next
    sections[1] by positions[..., 1] and so on, the rest passes through; freqs = rotary_frequencies(sections).  Positions and freqs have no
    gradient (refused if they require one).  -> (q', k'), or q' if k is None."""
    _no_tangent("rotary", q, k, positions, freqs)
    _constant("rotary: positions and freqs", positions.requires_grad or freqs.requires_grad)
    sections = tuple(int(s) for s in sections)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RotaryFn.apply(q, k, positions, freqs, sections, bool(interleaved))
    qo, ko = rotate(q, k, positions, freqs, sections, interleaved)
    return qo if k is None else (qo, ko)


# ---- attention --------------------------------------------------------------------------------------------------------------------
def _attention_args(q, k, v, mask, scale):
    dtype = _check("attention", q, k, v)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise RuntimeError(f"tatt_amd attention: q [B, Lq, H, D] and k, v [B, Lk, Hk, D] expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    _int("attention", B, Lq, Lk, H, Hk)
    if not 0 < D <= 128:
        raise NotImplementedError(f"tatt_amd attention: heads of 1 to 128 dimensions, got {D}")
    if Hk == 0 or H == 0 or H % Hk:
        raise RuntimeError(f"tatt_amd attention: {H} query heads are no multiple of {Hk} key heads")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != (B, Lk) or mask.device != q.device):
        raise RuntimeError(f"tatt_amd attention: key_padding_mask is a bool tensor [{B}, {Lk}] on q's device (True = leave the key out), got {tuple(mask.shape)} {mask.dtype} on {mask.device}")
    return dtype, (B, Lq, Lk, H, Hk, D), D ** -0.5 if scale is None else float(scale)


def _laid_out(t, dtype, group=1):
    """t as the kernels read it: rows of whole 16 bytes at 16-byte borders, a tile of 128 (of `group` heads) within 31-bit offsets; a copy, its rows
    padded with zeros (which add nothing to a product), if t is not."""
    sb, sl, sh, sd = t.stride()
    per = 8 if dtype else 4
    D = t.shape[3]
    if sd == 1 and D % per == 0 and sb % per == 0 and sl % per == 0 and sh % per == 0 and t.data_ptr() % 16 == 0 and (128 // group + 2) * sl + (group - 1) * sh <= 1 << 28:
        return t
    if D % per:
        return torch.nn.functional.pad(t, (0, -D % per)).contiguous()
    return t.clone(memory_format=torch.contiguous_format)


def attention_forward(q, k, v, key_padding_mask=None, causal=False, scale=None, need_saved=True):
    """-> (out, saved): `attention` without autograd; saved = (lse, low) is what attention_backward recomputes from (None unless need_saved): lse
    [B, H, Lq] fp32, the base-2 logarithm of each row's sum of exponentials (+inf where it sees nothing), and, for bfloat16, what rounding took from
    out (None for float32)."""
    dtype, dims, scale = _attention_args(q, k, v, key_padding_mask, scale)
    B, Lq, Lk, H, Hk, D = dims
    if B == 0 or Lq == 0 or Lk == 0:
        return q.new_zeros(q.shape), (q.new_full((B, H, Lq), float("inf"), dtype=torch.float32), None) if need_saved else None
    q, k, v = _laid_out(q, dtype, H // Hk), _laid_out(k, dtype), _laid_out(v, dtype)
    P = q.shape[3]
    dims = (B, Lq, Lk, H, Hk, P)
    out = _like(q)
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=q.device) if need_saved else None
    low = _like(q) if need_saved and dtype else None
    n = lib().cdll.tatt_mha_fwd_workspace(*dims, dtype)
    ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    mask_strides = None if key_padding_mask is None else _L2(*key_padding_mask.stride())
    _call("tatt_mha_fwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), _L9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]),
          _ptr(key_padding_mask), mask_strides, out.data_ptr(), _ptr(low), _ptr(lse), *dims, scale, bool(causal), dtype, _ptr(ws))
    return out if P == D else out[..., :D].contiguous(), (lse, low) if need_saved else None


def attention_backward(dout, q, k, v, out, saved, key_padding_mask=None, causal=False, scale=None):
    """-> (dq, dk, dv) of attention_forward with the same arguments: the probabilities are recomputed from what it saved."""
    dtype, dims, scale = _attention_args(q, k, v, key_padding_mask, scale)
    _check("attention", q, out, dout)
    B, Lq, Lk, H, Hk, D = dims
    lse, low = saved
    P = D + -D % (8 if dtype else 4)
    if (out.shape != q.shape or dout.shape != q.shape or lse.shape != (B, H, Lq) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous()
            or low is not None and (low.shape != (B, Lq, H, P) or low.dtype != torch.bfloat16 or not dtype or low.device != q.device or not low.is_contiguous())):
        raise RuntimeError("tatt_amd attention_backward: out and dout have the shape of q, saved is attention_forward's")
    if B == 0 or Lq == 0 or Lk == 0:
        return q.new_zeros(q.shape), k.new_zeros(k.shape), v.new_zeros(v.shape)
    q, out, dout = (_laid_out(t, dtype, H // Hk) for t in (q, out, dout))
    k, v = _laid_out(k, dtype), _laid_out(v, dtype)
    dims = (B, Lq, Lk, H, Hk, P)
    dq, dk, dv = _like(q), _like(k), _like(v)
    ws = torch.empty(lib().cdll.tatt_mha_bwd_workspace(*dims, dtype), dtype=torch.float32, device=q.device)
    mask_strides = None if key_padding_mask is None else _L2(*key_padding_mask.stride())
    _call("tatt_mha_bwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          _L15(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *dout.stride()[:3]), _ptr(key_padding_mask), mask_strides,
          out.data_ptr(), _ptr(low), dout.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dims, scale, bool(causal), dtype,
          ws.data_ptr())
    return (dq, dk, dv) if P == D else tuple(t[..., :D].contiguous() for t in (dq, dk, dv))


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, causal, scale):
        out, saved = attention_forward(q, k, v, mask, causal, scale)
        ctx.save_for_backward(q, k, v, out, *saved, mask)
        ctx.how = (causal, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        _first_order("attention")
        q, k, v, out, lse, low, mask = ctx.saved_tensors
        return (*attention_backward(dout, q, k, v, out, (lse, low), mask, *ctx.how), None, None, None)


def attention(q, k, v, key_padding_mask=None, causal=False, scale=None):
    """softmax(scale q k^T) v per head, the scores never in memory.  q [B, Lq, H, D], k and v [B, Lk, Hk, D] (float32 or bfloat16, any
    strides, D <= 128), H a multiple of Hk: query head h reads key head h // (H // Hk).  key_padding_mask [B, Lk] bool, True = leave the key out (as
    nn.MultiheadAttention's): nothing of such a key reaches a result.  causal: query i sees keys j <= i + Lk - Lq.  scale: D ** -0.5 if None.  A row
    that sees no key gives zeros and takes no part in any gradient.  No dropout.  -> out [B, Lq, H, D].

    What is not masked is expected to be finite: an infinity or NaN spreads to what a matrix product with it would reach, the rows from which only
    causality hides it included (0 times it).  float32 keeps its accuracy for magnitudes of 2^-100 to 2^127, scores (scaled) for magnitudes below
    2^28, past which a row may be NaN; the gradients' probabilities are off by 2^-24 of the score, relative to themselves."""
    _no_tangent("attention", q, k, v, scale)
    _constant("attention: scale", isinstance(scale, torch.Tensor) and scale.requires_grad)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFn.apply(q, k, v, key_padding_mask, causal, scale)
    return attention_forward(q, k, v, key_padding_mask, causal, scale, need_saved=False)[0]
