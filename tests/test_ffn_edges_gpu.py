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
