"""Microscaled 4-bit floating point (MXFP4 of the OCP Microscaling Formats specification, version 1.0).

A matrix is held as E2M1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), and every 32 of them along the contraction dim
share one E8M0 scale, a power of two.  With ``amax`` the largest magnitude of the 32,

    scale = 2^clamp(floor(log2 amax) - 2, -127, 127)        value = nearest E2M1 number to x / scale, ties to the even code, at most 6

so that a rounded value and all products of two are exact in fp32, and 17 bytes hold 32 values.  A block with an infinity or a NaN has
the scale code 255 and reads as NaN.

Layout of a matrix ``[R, K]`` (or of a stack ``[E, R, K]``, matrix by matrix), ``Kp`` = K rounded up to whole blocks:

* codes ``[R, Kp / 2]`` uint8: value 2i of a row in the low half of byte i, value 2i + 1 in the high half; zeros past K;
* scales ``[ceil(R / 128), ceil(Kp / 128), 512]`` uint8: biased exponents in tiles of 128 rows x 4 blocks, the order in which the tensor
  cores read them: row r, block j lies at ``[r / 128, j / 4, (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4]``; 127 (2^0) past the matrix.

Operators (``apb200::``; the functions below them check arguments and fill in defaults)

    mx4_quantize(x)                                  codes and scales of ``x`` [R, K] or [E, R, K]; blocks along the last dim
    mx4_dequantize(codes, scales, k, dtype)          the values they stand for
    mx4_round(x, dim)                                the same without the codes: ``x``, blocks along ``dim`` (the last, or the one before)
    mx4_mm(a, sa, b, sb, dtype)                      a [.., M, K] x b [.., N, K] -> [.., M, N], sums in fp32
    mx4_linear(x, codes, scales, dtype)              activations (rounded on the way) by weights held in 4 bits; gradient of ``x``
    mx4_matmul(x, w, trans_b, dtype)                 both operands rounded on the way; gradients of both
    mx4_mm_values(a, codes, scales, k, dtype)        a [.., N] (16 or 32 bits) by the values [N, k] of codes: gradients of ``x`` above; has
                                                     a gradient of ``a``

The rounding has no useful derivative; gradients go straight through it: with ``q`` for rounding and ``y = q(x) q(w)^T``,
``dx = dy q(w)`` and ``dw = dy^T q(x)``, products of the framework (``mm_nd``, ``grouped_mm``, ``mm_wgrad``): its own GEMM for bf16
operands, a library product, counted as such, for fp32 ones.  ``mx4_linear`` has second derivatives too; on CUDA ``mx4_matmul``, which keeps
its operands in 4 bits alone, refuses them.

The planner shards ``mx4_matmul`` like ``mm_nd`` / ``grouped_mm``; a contraction is split only into whole blocks.  The reference has no
4-bit formats; its float8 products are the nearest thing (autoparallel/graph_passes/async_tp/asynctp_ops.py:363-393).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .library import _ag, _make_cuda_entry, lib, ops, reference_impls

BLOCK = 32
TILE_ROWS, TILE_BLOCKS = 128, 4
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

lib.define("mx4_quantize(Tensor x) -> (Tensor, Tensor)")
lib.define("mx4_dequantize(Tensor codes, Tensor scales, int k, ScalarType dtype) -> Tensor")
lib.define("mx4_round(Tensor x, int dim) -> Tensor")
lib.define("mx4_mm(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, ScalarType out_dtype) -> Tensor")
lib.define("mx4_linear(Tensor x, Tensor codes, Tensor scales, ScalarType out_dtype) -> Tensor")
lib.define("mx4_matmul(Tensor x, Tensor w, bool trans_b, ScalarType out_dtype) -> Tensor")
lib.define("mx4_mm_values(Tensor a, Tensor codes, Tensor scales, int k, ScalarType out_dtype) -> Tensor")


def padded(k: int) -> int:
    """``k`` rounded up to whole blocks."""
    return (k + BLOCK - 1) // BLOCK * BLOCK


def scale_shape(rows: int, k: int) -> tuple[int, int, int]:
    return (rows + TILE_ROWS - 1) // TILE_ROWS, (k + BLOCK * TILE_BLOCKS - 1) // (BLOCK * TILE_BLOCKS), TILE_ROWS * TILE_BLOCKS


# ------------------------------------------------------------------------------------ references
def _pow2(n):
    """2^n as fp32 for -127 <= n <= 127, exactly."""
    n = n.to(torch.int32)
    return torch.where(n > -127, (n + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _blocks(x):
    """(codes [.., Kp], one a byte; biased exponents [.., Kp / 32]) of the last dim."""
    xf = F.pad(x.float(), (0, padded(x.shape[-1]) - x.shape[-1])).unflatten(-1, (-1, BLOCK))
    bits = (xf.contiguous().view(torch.int32) & 0x7FFFFFFF).amax(-1)  # (as integers: a NaN is larger than everything)
    field = bits >> 23
    broken = field == 255
    exponent = (field - 2).clamp_min(0)
    v = xf.abs() * _pow2(127 - exponent).unsqueeze(-1)
    code = (v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0)
    code = (code + 8 * torch.signbit(xf)).masked_fill(broken.unsqueeze(-1), 0)
    return code.flatten(-2).to(torch.uint8), torch.where(broken, 255, exponent).to(torch.uint8)


def _values(code, exponent):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=code.device)
    scale = _pow2(exponent.int().clamp_max(254) - 127).masked_fill(exponent == 255, float("nan"))
    return (table[code.long()].unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def tile_scales(exponent):
    """Biased exponents [.., R, K / 32] in the order of the layout."""
    r, j = exponent.shape[-2:]
    e = F.pad(exponent, (0, -j % TILE_BLOCKS, 0, -r % TILE_ROWS), value=127)
    e = e.unflatten(-2, (-1, 4, 32)).unflatten(-1, (-1, TILE_BLOCKS))  # [.., R / 128, 4, 32, tiles, 4]
    e = e.movedim(-2, -4).transpose(-2, -3)
    return e.reshape(*e.shape[:-3], TILE_ROWS * TILE_BLOCKS).contiguous()


def untile_scales(scales, rows: int, blocks: int):
    e = scales.unflatten(-1, (32, 4, TILE_BLOCKS)).transpose(-2, -3).movedim(-4, -2)
    return e.flatten(-2).flatten(-4, -2)[..., :rows, :blocks]


def _quantize(x):
    code, exponent = _blocks(x)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), tile_scales(exponent)


def _dequantize(codes, scales, k, dtype):
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return _values(code, untile_scales(scales, codes.shape[-2], codes.shape[-1] // 16))[..., :k].to(dtype)


def _round(x, dim):
    if dim == -2:
        return _round(x.transpose(-1, -2), -1).transpose(-1, -2).contiguous()
    return _values(*_blocks(x))[..., : x.shape[-1]].to(x.dtype).contiguous()


def _mm(a, a_scales, b, b_scales, out_dtype):
    k = 2 * a.shape[-1]
    av, bv = _dequantize(a, a_scales, k, torch.float32), _dequantize(b, b_scales, k, torch.float32)
    return torch.matmul(av, bv.transpose(-1, -2)).to(out_dtype)


def _linear(x, codes, scales, out_dtype):
    w = _dequantize(codes, scales, x.shape[-1], torch.float32)
    return torch.matmul(_round(x, -1).float(), w.transpose(-1, -2)).to(out_dtype)


def _matmul(x, w, trans_b, out_dtype):
    wq = _round(w, -1 if trans_b else -2).float()
    return torch.matmul(_round(x, -1).float(), wq.transpose(-1, -2) if trans_b else wq).to(out_dtype)


def _mm_values(a, codes, scales, k, out_dtype):
    return torch.matmul(a.float(), _dequantize(codes, scales, k, torch.float32)).to(out_dtype)


def _u8(x, *shape):
    return x.new_empty(shape, dtype=torch.uint8)


_REFS = {"mx4_quantize": _quantize, "mx4_dequantize": _dequantize, "mx4_round": _round, "mx4_mm": _mm, "mx4_linear": _linear,
         "mx4_matmul": _matmul, "mx4_mm_values": _mm_values}
_META = {
    "mx4_quantize": lambda x: (_u8(x, *x.shape[:-1], padded(x.shape[-1]) // 2),
                               _u8(x, *x.shape[:-2], *scale_shape(x.shape[-2], x.shape[-1]))),
    "mx4_dequantize": lambda codes, scales, k, dtype: codes.new_empty((*codes.shape[:-1], k), dtype=dtype),
    "mx4_round": lambda x, dim: x.new_empty(x.shape),
    "mx4_mm": lambda a, sa, b, sb, dtype: a.new_empty((*a.shape[:-1], b.shape[-2]), dtype=dtype),
    "mx4_linear": lambda x, codes, scales, dtype: x.new_empty((*x.shape[:-1], codes.shape[-2]), dtype=dtype),
    "mx4_mm_values": lambda a, codes, scales, k, dtype: a.new_empty((*a.shape[:-1], k), dtype=dtype),
    "mx4_matmul": lambda x, w, trans_b, dtype: x.new_empty((*x.shape[:-1], w.shape[-2 if trans_b else -1]), dtype=dtype),
}
for _name, _fn in _REFS.items():
    lib.impl(_name, _fn, "CPU")
    lib.impl(_name, _META[_name], "Meta")
    lib.impl(_name, _make_cuda_entry(_name), "CUDA")
    reference_impls[_name] = _fn


# ------------------------------------------------------------------------------------ autograd
def _pad8(t, *dims):
    """Zeros to multiples of 8 along ``dims``: the 16-bit products address rows of whole 16 bytes."""
    for d in dims:
        extra = -t.shape[d] % 8
        if extra:
            shape = list(t.shape)
            shape[d] = extra
            t = torch.cat((t, t.new_zeros(shape)), d)
    return t


def _times(a, b, trans_b, dtype):
    return ops.grouped_mm(a, b, trans_b, dtype) if b.ndim == 3 else ops.mm_nd(a, b, trans_b, dtype)


def _wgrad(a, b, grouped, dtype):
    return ops.grouped_mm_wgrad(a, b, dtype) if grouped else ops.mm_wgrad(a, b, dtype)


def _linear_setup(ctx, inputs, output):
    x, codes, scales, _ = inputs
    ctx.save_for_backward(codes, scales)
    ctx.k, ctx.dtype = x.shape[-1], x.dtype


def _linear_bwd(ctx, dy):
    codes, scales = ctx.saved_tensors
    return ops.mx4_mm_values(dy, codes, scales, ctx.k, ctx.dtype), None, None, None


def _matmul_setup(ctx, inputs, output):
    x, w, trans_b, _ = inputs
    ctx.save_for_backward(x, w)
    ctx.trans_b = trans_b


def _matmul_bwd(ctx, dy):
    x, w = ctx.saved_tensors
    tb, grouped = ctx.trans_b, w.ndim == 3
    if x.shape[-1] == 0 or dy.shape[-1] == 0:  # (the products take no matrices without columns)
        return torch.zeros_like(x), torch.zeros_like(w), None, None
    dyp = _pad8(dy, -1)
    dx = dw = None
    if ctx.needs_input_grad[0]:
        wq = _pad8(ops.mx4_round(w, -1 if tb else -2).to(dy.dtype), -1, -2)
        dx = _times(dyp, wq, not tb, x.dtype)
        dx = dx[..., : x.shape[-1]] if dx.shape[-1] != x.shape[-1] else dx
    if ctx.needs_input_grad[1]:
        xq = _pad8(ops.mx4_round(x, -1).to(dy.dtype), -1)
        dw = _wgrad(dyp, xq, grouped, w.dtype) if tb else _wgrad(xq, dyp, grouped, w.dtype)
        if dw.shape != w.shape:
            dw = dw[..., : w.shape[-2], : w.shape[-1]]
    return dx, dw, None, None


def _values_setup(ctx, inputs, output):
    a, codes, scales, k, _ = inputs
    ctx.save_for_backward(codes, scales)
    ctx.k, ctx.dtype = k, a.dtype


def _values_bwd(ctx, dc):
    codes, scales = ctx.saved_tensors
    n, k8 = codes.shape[-2], -(-ctx.k // 8) * 8
    if n == 0 or k8 == 0:
        return dc.new_zeros((*dc.shape[:-1], n), dtype=ctx.dtype), None, None, None, None
    w = _pad8(ops.mx4_dequantize(codes, scales, k8, dc.dtype), -2)
    da = _times(_pad8(dc, -1), w, True, ctx.dtype)
    return (da[..., :n] if da.shape[-1] != n else da), None, None, None, None


_ag("mx4_mm_values", _values_bwd, _values_setup)
_ag("mx4_linear", _linear_bwd, _linear_setup)
_ag("mx4_matmul", _matmul_bwd, _matmul_setup)
_ag("mx4_round", lambda ctx, dy: (dy, None), lambda ctx, inputs, output: None)


# ------------------------------------------------------------------------------------ Python API
_FLOATS = (torch.bfloat16, torch.float32)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check_float(name, **tensors):
    for key, t in tensors.items():
        _need(t.dtype in _FLOATS, f"{name}: {key} is {t.dtype}; bf16 or fp32 expected")


def _are_codes(codes, scales) -> bool:
    cs = codes.shape
    return (codes.dtype is scales.dtype is torch.uint8 and 2 <= len(cs) <= 3 and cs[-1] % 16 == 0
            and scales.shape == (*cs[:-2], (cs[-2] + 127) // 128, (cs[-1] + 63) // 64, 512))


def _check_codes(name, codes, scales):
    _need(codes.dtype == torch.uint8 and scales.dtype == torch.uint8, f"{name}: codes and scales are uint8")
    _need(codes.ndim in (2, 3) and codes.shape[-1] % 16 == 0,
          f"{name}: codes [R, Kp / 2] or [E, R, Kp / 2] of whole blocks, not {tuple(codes.shape)}")
    want = (*codes.shape[:-2], *scale_shape(codes.shape[-2], 2 * codes.shape[-1]))
    _need(tuple(scales.shape) == want,
          f"{name}: scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)} (expected {want})")


def _out_dtype(name, dtype, default):
    dtype = dtype or default
    _need(dtype in _FLOATS, f"{name}: a result of {dtype} is not offered (bf16 or fp32)")
    return dtype


def mx4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of ``x`` [R, K] or [E, R, K]; blocks along the last dim, whose stride may also be that of a transposed matrix."""
    if not (x.dtype in _FLOATS and 2 <= x.ndim <= 3):
        _check_float("mx4_quantize", x=x)
        _need(False, f"mx4_quantize: a matrix or a stack of matrices, not {x.ndim} dims")
    return ops.mx4_quantize(x)


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, k: int | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of codes and scales; ``k``: columns (default: whole blocks)."""
    cs = codes.shape
    k = 2 * cs[-1] if k is None else k
    if not (_are_codes(codes, scales) and (k + 31) // 32 * 16 == cs[-1] and dtype in _FLOATS):
        _check_codes("mx4_dequantize", codes, scales)
        _need(padded(k) == 2 * cs[-1], f"mx4_dequantize: {k} columns do not belong to {cs[-1]} bytes a row")
        _out_dtype("mx4_dequantize", dtype, None)
    return ops.mx4_dequantize(codes, scales, k, dtype)


def mx4_round(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    """``x`` with every 32 values along ``dim`` (the last dim, or the one before) rounded to 4 bits; its gradient goes straight through."""
    _check_float("mx4_round", x=x)
    _need(x.ndim >= 1 and dim in (-1, x.ndim - 1) or x.ndim >= 2 and dim in (-2, x.ndim - 2), f"mx4_round: dim {dim} of {x.ndim} dims")
    return ops.mx4_round(x, -1 if dim in (-1, x.ndim - 1) else -2)


def mx4_mm(a, a_scales, b, b_scales, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a`` [M, K] times the transpose of ``b`` [N, K], both in 4 bits; stacks [E, M, K] and [E, N, K] matrix by matrix."""
    _check_codes("mx4_mm", a, a_scales)
    _check_codes("mx4_mm", b, b_scales)
    _need(a.ndim == b.ndim and a.shape[-1] == b.shape[-1] and a.shape[:-2] == b.shape[:-2],
          f"mx4_mm: {tuple(a.shape)} and {tuple(b.shape)} do not multiply")
    return ops.mx4_mm(a, a_scales, b, b_scales, _out_dtype("mx4_mm", out_dtype, None))


def mx4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x`` [.., K] (rounded to 4 bits on the way) by weights ``mx4_quantize(w)`` of ``w`` [N, K] -> [.., N]; with weights of experts
    [E, N, K], ``x`` [E, M, K] -> [E, M, N].  The result has ``x``'s type unless another is asked for."""
    dtype = out_dtype or x.dtype
    xs, cs = x.shape, codes.shape
    # (one test for the calls that are right: this is the path of single tokens)
    if not (x.dtype in _FLOATS and dtype in _FLOATS and _are_codes(codes, scales) and xs and (xs[-1] + 31) // 32 * 16 == cs[-1]
            and (len(cs) == 2 or (len(xs) == 3 and xs[0] == cs[0]))):
        _check_float("mx4_linear", x=x)
        _check_codes("mx4_linear", codes, scales)
        _need(x.ndim >= 1 and padded(xs[-1]) == 2 * cs[-1], f"mx4_linear: x {tuple(xs)} and codes {tuple(cs)} do not multiply")
        _need(codes.ndim == 2 or (x.ndim == 3 and xs[0] == cs[0]),
              f"mx4_linear: weights of {cs[0]} experts take x [E, M, K], not {tuple(xs)}")
        _out_dtype("mx4_linear", dtype, None)
    return ops.mx4_linear(x, codes, scales, dtype)


def mx4_mm_values(a: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, k: int | None = None,
                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``a`` [.., N] by the values [N, k] that codes and scales stand for -> [.., k]; with a stack of codes [E, N, ..], ``a``
    [E, M, N] -> [E, M, k]."""
    _check_float("mx4_mm_values", a=a)
    _check_codes("mx4_mm_values", codes, scales)
    k = 2 * codes.shape[-1] if k is None else k
    _need(padded(k) == 2 * codes.shape[-1], f"mx4_mm_values: {k} columns do not belong to {codes.shape[-1]} bytes a row")
    _need(a.ndim >= 1 and a.shape[-1] == codes.shape[-2] and (codes.ndim == 2 or a.ndim == 3 and a.shape[0] == codes.shape[0]),
          f"mx4_mm_values: a {tuple(a.shape)} and codes {tuple(codes.shape)} do not multiply")
    return ops.mx4_mm_values(a, codes, scales, k, _out_dtype("mx4_mm_values", out_dtype, a.dtype))


def mx4_matmul(x: torch.Tensor, w: torch.Tensor, trans_b: bool = True, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x`` [.., K] by ``w`` ([N, K] if ``trans_b`` else [K, N]), or ``x`` [E, M, K] by ``w`` [E, N, K] / [E, K, N], both rounded to 4 bits
    on the way in blocks along K."""
    dtype = out_dtype or x.dtype
    xs, ws = x.shape, w.shape
    fits = xs and (len(ws) == 2 or (len(ws) == len(xs) == 3 and xs[0] == ws[0])) and xs[-1] == ws[-1 if trans_b else -2]
    if not (fits and x.dtype in _FLOATS and w.dtype in _FLOATS and dtype in _FLOATS):
        _check_float("mx4_matmul", x=x, w=w)
        _need(fits, f"mx4_matmul: x {tuple(xs)}, w {tuple(ws)}: [.., K] by a matrix, or [E, M, K] by a stack, of the same K")
        _out_dtype("mx4_matmul", dtype, None)
    return ops.mx4_matmul(x, w, trans_b, dtype)
