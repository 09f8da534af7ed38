"""The feed-forward half of a decoder layer with its ends fused, and activations that are held in 8 bits.

Operators (``apb200::``; the functions at the end of this file check arguments and fill in defaults)

    add_rms_norm(x, residual, weight, eps)        h = x + residual (rounded to its type) and y = rms_norm(h)
    add_rms_norm_fp8(.., keep)                    the same with y in e4m3, one scale a row, as ``scaled_mm`` takes them; the residual may
                                                  be left out
    gated_ffn(x, w1, w3, w2, act, bits)           (act(x w1^T) * (x w3^T)) w2^T
    mx8_quantize(x), mx8_dequantize(..)           activations in 8 bits

and what the gradients of the block are made with: ``add_rms_norm_bwd``, ``gated_mm`` (both projections and their product),
``gated_dgrad`` (through w2 and the product), ``gated_dx``, ``gated_wgrad``.

Norm.  With ``r = 1 / sqrt(mean(h^2) + eps)``, ``n = h r``, ``g = dy w``:

    y = n w        dx = dresidual = dh + r (g - n mean(g n))        dw = sum over rows of dy n

and in 8 bits ``scale = max |y| / 448`` (1 for a row whose maximum is below 2^-100), ``q = e4m3(y / scale)``.

Gated block.  With ``a = x w1^T``, ``b = x w3^T``, ``h = act(a) * b``, ``y = h w2^T``:

    dh = dy w2       da = dh b act'(a)       db = dh act(a)
    dx = da w1 + db w3       dw1 = da^T x       dw3 = db^T x       dw2 = dy^T h

a and b are kept for the backward pass, ``ab`` [.., 2, H], h is made again from them.  ``bits`` 11 keeps x as it is, and a, b as fp16 numbers
under a power of two (below) where x is bf16, as they are where it is fp32; 16 the same with 16-bit codes; 8 keeps all three as 8-bit
checkpoints, from which all gradients are made; 0 keeps nothing (no gradients).  da, db and the h of the backward pass are rounded to x's type, which is what the products of the
gradients take.

8-bit checkpoints (MXINT8 of the OCP Microscaling Formats specification, version 1.0).  32 values along the last dim share a power of two,

    e = max(floor(log2 of the largest magnitude), -120)     code = v 2^(6-e), rounded to even, within +-127     value = code 2^(e-6)

codes int8 of the values' shape, scales uint8 [.., ceil(K / 32)]: e + 127, and 255 for a block with an infinity or a NaN, which reads as
NaN.  (The format's e goes down to -127.  What is written here stops at -120, where the unit is the smallest normal fp32 number; what is read
may have any scale.)  A value is off by at most 2^(e-7), but 2^(e-6) where it is the block's largest and rounds to 128; it is exact in bf16.  The 16-bit
codes are the same with 14 for 6, -112 for -120 and 32767 for 127: in as many bits as bf16, off by 2^-15 of the block's largest value and
not by 2^-8 of each, which is more where that is 128 times the value.  fp16 numbers, v 2^(14-e) with the same e and scales, keep a value's own
exponent: off by at most 2^-11 of it down to 2^-28 of the block's largest, and by 2^-39 of that below.

The reference leaves these to the tracing compiler (``x + attention``, RMSNorm and SwiGLU of
autoparallel/_testing/models/llama3.py:320-429); it has no 8-bit checkpoints.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .library import _ag, _make_cuda_entry, _rms_norm_bwd_ref, _rms_norm_ref, lib, ops, reference_impls

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
CHECKPOINTS = {"full": 11, "mx16": 16, "mx8": 8}
BLOCK = 32
_CODES = {8: torch.int8, 11: torch.float16, 16: torch.int16}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0

lib.define("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)")
lib.define("add_rms_norm_bwd(Tensor dy, Tensor? dh, Tensor h, Tensor weight, Tensor rstd) -> (Tensor, Tensor)")
lib.define("add_rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps, bool keep) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
lib.define("mx8_quantize(Tensor x) -> (Tensor, Tensor)")
lib.define("mx8_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor")
lib.define("gated_mm(Tensor x, Tensor w1, Tensor w3, int act, int bits) -> (Tensor, Tensor, Tensor)")
lib.define("gated_dgrad(Tensor dy, Tensor w2, Tensor ab, Tensor scales, int act) -> (Tensor, Tensor)")
lib.define("gated_dx(Tensor dab, Tensor w1, Tensor w3) -> Tensor")
lib.define("gated_wgrad(Tensor dab, Tensor x, ScalarType dtype) -> (Tensor, Tensor)")
lib.define("gated_ffn(Tensor x, Tensor w1, Tensor w3, Tensor w2, int act, int bits) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")


def mx8_blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


# ------------------------------------------------------------------------------------ references
def _add_rms_norm(x, residual, weight, eps):
    h = (x.float() + residual.float()).to(x.dtype)
    y, rstd = _rms_norm_ref(h, weight, eps)
    return y, h, rstd


def _add_rms_norm_bwd(dy, dh, h, weight, rstd):
    if dh is None:
        return _rms_norm_bwd_ref(dy, h, weight, rstd)
    n = h.float() * rstd.unsqueeze(-1)
    g = dy.float() * weight.float()
    dx = dh.float() + rstd.unsqueeze(-1) * (g - n * (g * n).mean(-1, keepdim=True))
    dw = (dy.float() * n).reshape(-1, h.shape[-1]).sum(0)
    return dx.to(h.dtype), dw.to(weight.dtype)


def _add_rms_norm_fp8(x, residual, weight, eps, keep):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    rstd = torch.rsqrt(h.float().pow(2).mean(-1, keepdim=True) + eps)
    y = h.float() * rstd * weight.float()
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.where(top < 2.0**-100, 1.0, top / F8_MAX)
    q = (y / scale).clamp(-F8_MAX, F8_MAX).to(F8)
    none = x.new_empty(0)
    return y.to(x.dtype) if keep else none, none.clone() if residual is None else h, rstd.squeeze(-1), q, scale


def _quantize(x, bits):
    k = x.shape[-1]
    v = F.pad(x.float(), (0, -k % BLOCK)).unflatten(-1, (mx8_blocks(k), BLOCK))
    field = (v.contiguous().view(torch.int32) & 0x7FFFFFFF).amax(-1) >> 23  # (as integers: a NaN is larger than everything)
    broken = field == 255
    n = 8 if bits == 8 else 16
    byte = field.clamp(min=n - 1)
    to_code = ((252 + n - byte).clamp(min=1) << 23).to(torch.int32).view(torch.float32).masked_fill(broken, 0.0)
    code = torch.nan_to_num(v * to_code.unsqueeze(-1), nan=0.0)
    if bits != 11:
        code = torch.round(code).clamp(1 - 2 ** (n - 1), 2 ** (n - 1) - 1)
    return code.flatten(-2)[..., :k].to(_CODES[bits]).contiguous(), byte.to(torch.uint8)


def _dequantize(codes, scales, dtype):
    s = scales.int()
    field = s + 2 - 8 * codes.element_size()  # (of the unit, 2^(field - 127); scales from elsewhere may go below 1)
    unit = torch.where(field > 0, field << 23, 0x400000 >> (-field).clamp(0, 31)).to(torch.int32).view(torch.float32).masked_fill(s == 255, float("nan"))
    return (codes.float() * unit.repeat_interleave(BLOCK, -1)[..., : codes.shape[-1]]).to(dtype)


def _mx8_quantize(x):
    return _quantize(x, 8)


_mx8_dequantize = _dequantize


def _act(act: int, a):
    """act(a) and its derivative, fp32."""
    if act == 1:
        phi = 0.5 * torch.erfc(a * -(0.5**0.5))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) * 0.3989422804014327
    if act == 0:
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    s = torch.sigmoid(1.5957691216057308 * a * (1 + 0.044715 * a * a))
    return a * s, s + a * s * (1 - s) * (1.5957691216057308 + 0.21406444881780073 * a * a)


def _kept(ab, bits, dtype):
    none = ab.new_empty(0, dtype=torch.uint8)
    if bits == 0:
        return ab.new_empty(0, dtype=dtype), none
    return (ab, none) if bits != 8 and dtype is torch.float32 else _quantize(ab, bits)


def _values(ab, scales):
    return ab if ab.dtype is torch.float32 else _dequantize(ab, scales, torch.float32)


def _gated_mm(x, w1, w3, act, bits):
    a, b = (torch.matmul(x.float(), w.float().t()) for w in (w1, w3))
    return ((_act(act, a)[0] * b).to(x.dtype), *_kept(torch.stack((a, b), -2), bits, x.dtype))


def _gated_dgrad(dy, w2, ab, scales, act):
    dh = torch.matmul(dy.float(), w2.float())
    a, b = _values(ab, scales).unbind(-2)
    g, d = _act(act, a)
    return torch.stack((dh * b * d, dh * g), -2).to(dy.dtype), (g * b).to(dy.dtype)


def _gated_dx(dab, w1, w3):
    da, db = dab.float().unbind(-2)
    return (torch.matmul(da, w1.float()) + torch.matmul(db, w3.float())).to(dab.dtype)


def _gated_wgrad(dab, x, dtype):
    rows = x.shape[:-1].numel()
    xf = x.float().reshape(rows, x.shape[-1])
    return tuple(torch.matmul(d.reshape(rows, d.shape[-1]).t(), xf).to(dtype) for d in dab.float().unbind(-2))


def _gated_ffn(x, w1, w3, w2, act, bits):
    h, ab, scales = _gated_mm(x, w1, w3, act, bits)
    y = torch.matmul(h.float(), w2.float().t()).to(x.dtype)
    none = x.new_empty(0, dtype=torch.uint8)
    return (y, ab, scales, *(_mx8_quantize(x) if bits == 8 else (none, none.clone())))


# ------------------------------------------------------------------------------------ meta
def _new(x, shape, dtype=None):
    return x.new_empty(shape, dtype=dtype or x.dtype)


def _kept_meta(x, lead, n, bits):
    """(ab, scales) for [.., n]"""
    if bits == 0 or (bits != 8 and x.dtype is torch.float32):
        return _new(x, (*lead, n) if bits else (0,)), _new(x, (0,), torch.uint8)
    return _new(x, (*lead, n), _CODES[bits]), _new(x, (*lead, mx8_blocks(n)), torch.uint8)


def _add_rms_norm_fp8_meta(x, residual, weight, eps, keep):
    lead = x.shape[:-1]
    return (_new(x, x.shape if keep else (0,)), _new(x, x.shape if residual is not None else (0,)), _new(x, lead, torch.float32),
            _new(x, x.shape, F8), _new(x, (*lead, 1), torch.float32))


def _gated_ffn_meta(x, w1, w3, w2, act, bits):
    lead = x.shape[:-1]
    xq = _kept_meta(x, lead, x.shape[-1], 8) if bits == 8 else (_new(x, (0,), torch.uint8), _new(x, (0,), torch.uint8))
    return (_new(x, (*lead, w2.shape[0])), *_kept_meta(x, (*lead, 2), w1.shape[0], bits), *xq)


_META = {
    "add_rms_norm": lambda x, residual, weight, eps: (_new(x, x.shape), _new(x, x.shape), _new(x, x.shape[:-1], torch.float32)),
    "add_rms_norm_bwd": lambda dy, dh, h, weight, rstd: (_new(h, h.shape), _new(weight, weight.shape)),
    "add_rms_norm_fp8": _add_rms_norm_fp8_meta,
    "mx8_quantize": lambda x: _kept_meta(x, x.shape[:-1], x.shape[-1], 8),
    "mx8_dequantize": lambda codes, scales, dtype: _new(codes, codes.shape, dtype),
    "gated_mm": lambda x, w1, w3, act, bits: (_new(x, (*x.shape[:-1], w1.shape[0])), *_kept_meta(x, (*x.shape[:-1], 2), w1.shape[0], bits)),
    "gated_dgrad": lambda dy, w2, ab, scales, act: (_new(dy, ab.shape), _new(dy, (*dy.shape[:-1], w2.shape[1]))),
    "gated_dx": lambda dab, w1, w3: _new(dab, (*dab.shape[:-2], w1.shape[1])),
    "gated_wgrad": lambda dab, x, dtype: tuple(_new(x, (dab.shape[-1], x.shape[-1]), dtype) for _ in range(2)),
    "gated_ffn": _gated_ffn_meta,
}
_REFS = {"add_rms_norm": _add_rms_norm, "add_rms_norm_bwd": _add_rms_norm_bwd, "add_rms_norm_fp8": _add_rms_norm_fp8,
         "mx8_quantize": _mx8_quantize, "mx8_dequantize": _mx8_dequantize, "gated_mm": _gated_mm, "gated_dgrad": _gated_dgrad,
         "gated_dx": _gated_dx, "gated_wgrad": _gated_wgrad, "gated_ffn": _gated_ffn}
for _name, _fn in _REFS.items():
    lib.impl(_name, _fn, "CPU")
    lib.impl(_name, _META[_name], "Meta")
    lib.impl(_name, _make_cuda_entry(_name), "CUDA")
    reference_impls[_name] = _fn


# ------------------------------------------------------------------------------------ autograd
def _norm_setup(ctx, inputs, output):
    ctx.save_for_backward(output[1], inputs[2], output[2])


def _norm_bwd(ctx, dy, dh, _drstd):
    dx, dw = ops.add_rms_norm_bwd(dy, dh, *ctx.saved_tensors)
    return dx, dx, dw, None


_ag("add_rms_norm", _norm_bwd, _norm_setup)


def _norm8_setup(ctx, inputs, output):
    x, residual, weight, _, keep = inputs
    ctx.residual = residual is not None
    ctx.save_for_backward(output[1] if ctx.residual else x, weight, output[2])
    ctx.mark_non_differentiable(output[2], output[3], output[4], *(() if keep else (output[0],)), *(() if ctx.residual else (output[1],)))


def _norm8_bwd(ctx, dy, dh, _drstd, _dq, _dscale):
    dx, dw = ops.add_rms_norm_bwd(dy, dh if ctx.residual else None, *ctx.saved_tensors)
    return dx, dx if ctx.residual else None, dw, None, None


_ag("add_rms_norm_fp8", _norm8_bwd, _norm8_setup)


def _ffn_setup(ctx, inputs, output):
    x, w1, w3, w2, act, bits = inputs
    _, ab, scales, xq, xs = output
    ctx.mark_non_differentiable(ab, scales, xq, xs)
    ctx.act, ctx.bits, ctx.dtype = act, bits, x.dtype
    ctx.save_for_backward(w1, w3, w2, ab, scales, *((xq, xs) if bits == 8 else (x,)))


def _ffn_bwd(ctx, dy, *_):
    if ctx.bits == 0:
        raise RuntimeError("gated_ffn: a call that kept nothing has no gradients")
    w1, w3, w2, ab, scales, *x = ctx.saved_tensors
    x = ops.mx8_dequantize(*x, ctx.dtype) if ctx.bits == 8 else x[0]
    dab, h = ops.gated_dgrad(dy, w2, ab, scales, ctx.act)
    dw2 = ops.mm_wgrad(dy, h, w2.dtype) if w2.numel() else torch.zeros_like(w2)  # (the products take no matrices without columns)
    dw1, dw3 = ops.gated_wgrad(dab, x, w1.dtype)
    return ops.gated_dx(dab, w1, w3), dw1, dw3, dw2, None, None


_ag("gated_ffn", _ffn_bwd, _ffn_setup)


# ------------------------------------------------------------------------------------ Python API
_FLOATS = (torch.bfloat16, torch.float32)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check_norm(name, x, residual, weight):
    _need(x.dtype in _FLOATS, f"{name}: x is {x.dtype}; bf16 or fp32 expected")
    _need(x.ndim >= 1 and x.shape[-1] >= 1, f"{name}: x [.., D] with D at least 1, not {tuple(x.shape)}")
    _need(x.shape[-1] <= 32768, f"{name}: rows of {x.shape[-1]} values; at most 32768")
    if residual is not None:
        _need(residual.shape == x.shape and residual.dtype == x.dtype,
              f"{name}: residual {tuple(residual.shape)} {residual.dtype} and x {tuple(x.shape)} {x.dtype} are not alike")
    _need(tuple(weight.shape) == (x.shape[-1],) and weight.dtype in _FLOATS,
          f"{name}: weight {tuple(weight.shape)} {weight.dtype}; [{x.shape[-1]}] in bf16 or fp32 expected")
    _need(weight.device == x.device and (residual is None or residual.device == x.device), f"{name}: operands on different devices")


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual``, rounded to their type, and ``rms_norm(h, weight)``: (norm, h).  Gradients of both results reach x, the
    residual and the weight in one pass.  (On CUDA a weight in fp32 beside bf16 operands is taken in bf16, as ``rms_norm`` takes it; its
    gradient is fp32.)"""
    xs = x.shape
    if not (x.dtype in _FLOATS and xs and 1 <= xs[-1] <= 32768 and residual.shape == xs and residual.dtype is x.dtype
            and weight.shape == xs[-1:] and weight.dtype in _FLOATS and x.device == residual.device == weight.device):
        _check_norm("add_rms_norm", x, residual, weight)
    y, h, _ = ops.add_rms_norm(x, residual, weight, eps)
    return y, h


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-5, keep: bool = True):
    """``add_rms_norm`` (of x alone where ``residual`` is None) with the norm in 8 bits: (y, h, q, scale), ``q`` float8_e4m3fn and
    ``scale`` fp32 [.., 1], the row-wise operands of ``scaled_mm``; ``q * scale`` stands for the norm.  q and scale have no gradient: a
    training step hands the gradient of what it made of them to ``y``, the norm itself, which ``keep=False`` leaves out (None)."""
    xs = x.shape
    # (one test for the calls that are right: this is the path of single tokens)
    if not (x.dtype in _FLOATS and xs and 1 <= xs[-1] <= 32768 and weight.shape == xs[-1:] and weight.dtype in _FLOATS
            and weight.device == x.device
            and (residual is None or (residual.shape == xs and residual.dtype is x.dtype and residual.device == x.device))):
        _check_norm("add_rms_norm_fp8", x, residual, weight)
    if not keep and torch.is_grad_enabled():
        _need(not any(t is not None and t.requires_grad for t in (x, residual, weight)),
              "add_rms_norm_fp8: gradients go through y, which keep=False leaves out")
    y, h, _, q, scale = ops.add_rms_norm_fp8(x, residual, weight, eps, keep)
    return y if keep else None, x if residual is None else h, q, scale


def mx8_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [.., K], scales uint8 [.., ceil(K / 32)]) of ``x`` [.., K]."""
    _need(x.dtype in _FLOATS, f"mx8_quantize: x is {x.dtype}; bf16 or fp32 expected")
    _need(x.ndim >= 1, "mx8_quantize: x has no dims")
    return ops.mx8_quantize(x)


def mx8_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of codes and scales, of any scale of the format, exact in both types that are offered (bf16, fp32; code -128 of the
    largest scale, -2^128, is -infinity)."""
    _need(codes.dtype is torch.int8 and scales.dtype is torch.uint8 and codes.ndim >= 1,
          f"mx8_dequantize: int8 codes and uint8 scales expected, not {codes.dtype} and {scales.dtype}")
    want = (*codes.shape[:-1], mx8_blocks(codes.shape[-1]))
    _need(tuple(scales.shape) == want and scales.device == codes.device,
          f"mx8_dequantize: scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)} (expected {want}, on their device)")
    _need(dtype in _FLOATS, f"mx8_dequantize: a result of {dtype} is not offered (bf16 or fp32)")
    return ops.mx8_dequantize(codes, scales, dtype)


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor, act: str = "silu",
              checkpoint: str = "full") -> torch.Tensor:
    """``(act(x w1^T) * (x w3^T)) w2^T``: x [.., D], w1 and w3 [H, D], w2 [N, H] -> [.., N].  ``act``: "silu", "gelu" (by the error
    function) or "gelu_tanh".  ``checkpoint``: what the backward pass finds, "full" (x, and both projections in as many bits as its type
    has, of bf16 to 2^-11 of each value), "mx16" (the same of bf16 as whole numbers, to 2^-15 of the largest of 32 neighbours) or "mx8" (all
    in 8 bits, about half the memory; the gradients are those of the rounded values)."""
    xs, ws = x.shape, w1.shape
    fits = (len(xs) >= 1 and len(ws) == 2 and w3.shape == ws and w2.ndim == 2 and ws[1] == xs[-1] and w2.shape[1] == ws[0]
            and x.dtype in _FLOATS and x.dtype is w1.dtype is w3.dtype is w2.dtype and x.device == w1.device == w3.device == w2.device)
    if not (fits and act in ACTS and checkpoint in CHECKPOINTS):
        _need(act in ACTS, f"gated_ffn: act is one of {sorted(ACTS)}, not {act!r}")
        _need(checkpoint in CHECKPOINTS, f"gated_ffn: checkpoint is one of {sorted(CHECKPOINTS)}, not {checkpoint!r}")
        _need(x.dtype in _FLOATS and x.dtype is w1.dtype is w3.dtype is w2.dtype,
              f"gated_ffn: x, w1, w3, w2 are {x.dtype}, {w1.dtype}, {w3.dtype}, {w2.dtype}; all bf16 or all fp32 expected")
        _need(x.device == w1.device == w3.device == w2.device, "gated_ffn: operands on different devices")
        _need(False, f"gated_ffn: x {tuple(xs)}, w1 {tuple(ws)}, w3 {tuple(w3.shape)}, w2 {tuple(w2.shape)}: "
                     "[.., D], [H, D], [H, D], [N, H] expected")
    records = torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w3.requires_grad or w2.requires_grad)
    return ops.gated_ffn(x, w1, w3, w2, ACTS[act], CHECKPOINTS[checkpoint] if records else 0)[0]
