"""The feed-forward operators where a first set of tests did not look: one of two results used, scales from elsewhere, blocks with a large value, rows
of unusual size.

Tolerances are relative to the size of the terms that a result is summed from; a rounding to a type is off by at most half a step of it."""
import math

import pytest
import torch
import torch.nn.functional as F

import autoparallel_b200.ops as K
from autoparallel_b200.ops import ffn_ops as FFN
from autoparallel_b200.ops.library import ops

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0**-8, F32: 2.0**-24}
ARITHMETIC = 16 * 2.0**-22  # of a norm's terms: 1 / rms by an instruction of 2^-22, sums in chains of a row's width / threads and a tree


@pytest.fixture(scope="module", autouse=True)
def loaded():
    from autoparallel_b200.ops import cuda_impl

    cuda_impl.ensure_loaded()
    yield cuda_impl
    cuda_impl.check_status()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, gen, dtype=BF, scale=1.0):
    return (scale * torch.randn(*shape, device="cuda", generator=gen)).to(dtype)


# ------------------------------------------------------------------------------------ norm
def _norm_gradients(h, w, dy, dh, eps):
    """(dx, dw) in 64 bits, and the sum of the magnitudes of each one's terms."""
    h, w, dy = h.double(), w.double(), dy.double()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    n, g = h * r, dy * w
    dh = torch.zeros_like(h) if dh is None else dh.double()
    dx = dh + r * (g - n * (g * n).mean(-1, keepdim=True))
    terms = dh.abs() + r * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    flat = (dy * n).reshape(-1, h.shape[-1])
    return dx, flat.sum(0), terms, flat.abs().sum(0)


def _check_norm_gradients(got, want, dtype, weight_dtype):
    dx, dw, terms, dw_terms = want
    assert bool(((got[0].double() - dx).abs() <= HALF_STEP[dtype] * dx.abs() + ARITHMETIC * terms).all())
    assert all(torch.equal(got[0], t) for t in got[1:-1])
    assert got[-1].dtype == weight_dtype
    # (a sum over rows: in chains of rows / blocks and a tree)
    assert bool(((got[-1].double() - dw).abs() <= HALF_STEP[weight_dtype] * dw.abs() + ARITHMETIC * dw_terms).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("form", ["norm", "fp8", "fp8 of x alone"])
@pytest.mark.parametrize("D", [1, 7, 8, 1001, 8191, 16384, 16392, 32767, 32768])
def test_gradients_where_only_the_norm_is_used(D, form, dtype):
    """Every width that the forward pass takes, in one row and in more rows than there are blocks of the smallest."""
    for rows in (1, 37) if D > 8 else (1, 37, 5000):
        g = _gen(D + rows)
        x, r, dy = (_randn(rows, D, gen=g, dtype=dtype) for _ in range(3))
        w = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dtype)
        if form == "fp8 of x alone":
            leaves, h = [t.clone().requires_grad_() for t in (x, w)], x
            y = K.add_rms_norm_fp8(leaves[0], None, leaves[1])[0]
        else:
            leaves, h = [t.clone().requires_grad_() for t in (x, r, w)], (x.float() + r.float()).to(dtype)
            y = (K.add_rms_norm if form == "norm" else K.add_rms_norm_fp8)(*leaves)[0]
        got = torch.autograd.grad(y, leaves, dy)
        _check_norm_gradients(got, _norm_gradients(h, w, dy, None, 1e-5), dtype, dtype)


# ------------------------------------------------------------------------------------ 8-bit checkpoints
@pytest.mark.parametrize("k", [256, 264, 257, 1003])
def test_mx8_values_of_every_scale(k):
    """Codes from elsewhere may come with any scale byte of the format, and with the code -128."""
    codes = (torch.arange(k, device="cuda") % 256 - 128).to(torch.int8).expand(256, k).contiguous()
    scales = torch.arange(256, device="cuda").to(torch.uint8).unsqueeze(1).expand(256, -(-k // 32)).contiguous()
    want = codes.double() * torch.exp2(scales[:, :1].double() - 133)
    want[255] = math.nan
    for dtype in (BF, F32):  # (exact in both but for -2^128)
        got = K.mx8_dequantize(codes, scales, dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[:255].double(), want[:255].masked_fill(want[:255] <= -(2.0**128), -math.inf))
        assert torch.equal(K.mx8_dequantize(codes.cpu(), scales.cpu(), dtype).nan_to_num(nan=3.0), got.cpu().nan_to_num(nan=3.0))
