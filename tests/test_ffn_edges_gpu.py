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


# ------------------------------------------------------------------------------------ gated block
@pytest.mark.parametrize("M,D,H", [(256, 128, 128), (300, 72, 1000), (2100, 256, 520), (40, 36, 100)])
@pytest.mark.parametrize("times", [1, 64, 4096, 2.0**15, 2.0**24])
def test_full_keeps_small_values_beside_large_ones(M, D, H, times):
    """One column of every block of 32 is much larger than the others; the gradients of the others' weights are as near to 64 bits as they are without it."""
    g = _gen(M)
    x, dy = _randn(M, D, gen=g), _randn(M, 64, gen=g)
    w1, w3, w2 = _randn(H, D, gen=g, scale=D**-0.5), _randn(H, D, gen=g, scale=D**-0.5), _randn(64, H, gen=g, scale=H**-0.5)
    large = torch.arange(H, device="cuda") % 32 == 5
    w1[large] *= times
    w3[large] *= times
    leaves = [t.requires_grad_() for t in (x, w1, w3, w2)]
    got = torch.autograd.grad(K.gated_ffn(*leaves), leaves, dy)
    d = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad((F.silu(d[0] @ d[1].t()) * (d[0] @ d[2].t())) @ d[3].t(), d, dy.double())
    for u, v in ((got[1][~large], want[1][~large]), (got[2][~large], want[2][~large]), (got[3][:, ~large], want[3][:, ~large])):
        # two roundings to bf16 (da, db or h, and the result), each at most 2^-8 and evenly spread: sqrt(2 / 3) 2^-8; what is kept adds 2^-11 of each value at most
        assert float((u.double() - v).norm() / v.norm()) <= math.sqrt(2 / 3) * 2.0**-8 + 2.0**-11


# rows: split kernel, single CTAs, pairs, wide pairs, the plain products; columns: parts of tiles and of blocks of 32
@pytest.mark.parametrize("M,D,H", [(1, 64, 8), (3, 256, 40), (17, 2048, 1408), (33, 64, 136), (130, 1288, 520), (300, 136, 2056), (999, 2048, 1408), (2100, 72, 1000), (4096, 4416, 1032),
                                   (20, 60, 64), (37, 64, 63)])
def test_fp16_numbers_of_both_projections(M, D, H):
    act = ("silu", "gelu", "gelu_tanh")[(M + D + H) % 3]
    fn = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act]
    g = _gen(M)
    x, dy = _randn(M, D, gen=g), _randn(M, 128, gen=g)
    # columns of very different sizes within a block
    w1, w3 = ((_randn(H, D, gen=g, dtype=F32, scale=D**-0.5) * torch.exp2(torch.randint(-20, 1, (H, 1), device="cuda", generator=g).float())).to(BF) for _ in range(2))
    w2 = _randn(128, H, gen=g, scale=H**-0.5)
    h, ab, scales = ops.gated_mm(x, w1, w3, FFN.ACTS[act], 11)
    assert ab.dtype == torch.float16 and ab.shape == (M, 2, H) and scales.shape == (M, 2, -(-H // 32)) and bool((scales >= 15).all())
    exact = torch.stack([x.double() @ w.double().t() for w in (w1, w3)], 1)
    kept = ab.double() * torch.exp2(scales.double() - 141).repeat_interleave(32, -1)[..., :H]
    # fp16's half step, and the products' own error: a step of 16 terms rounds the accumulator, which may cut it off (2^-23 and not a half of that), at its running
    # size; that is a partial sum of independent terms with random signs, so within 6 times the root of the sum of their squares (normal: 2e-9 of all are not)
    acc = (D / 16 + 1) * 2.0**-23 * 6 * torch.stack([(x.double().square() @ w.double().square().t()).sqrt() for w in (w1, w3)], 1)
    off = (kept - exact).abs() - 2.0**-11 * exact.abs()
    assert bool((off <= 1.01 * acc).all()), float((off / acc).max())
    dab, h2 = ops.gated_dgrad(dy, w2, ab, scales, FFN.ACTS[act])
    a, b = (t.clone().requires_grad_() for t in kept.unbind(1))
    hd = fn(a) * b
    dh = dy.double() @ w2.double()
    da, db = torch.autograd.grad(hd, (a, b), dh)
    hd, a, b = hd.detach(), a.detach(), b.detach()
    # a half step of bf16; of dh: the terms' sum in fp32; of the activation and its derivative: 2^-18 of their terms (|act| <= |a|, |act'| <= 1.13 for all three)
    off = (128 / 16 + 1) * 2.0**-23 * 6 * (dy.double().square() @ w2.double().square()).sqrt()
    for got, want, slope in ((dab[:, 0], da, 1.13 * b.abs()), (dab[:, 1], db, a.abs())):
        assert bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 1.01 * (off + 2.0**-18 * dh.abs()) * slope).all())
    assert bool(((h2.double() - hd).abs() <= (2.0**-8 + 2.0**-17) * hd.abs() + 2.0**-140).all())


def test_fp16_numbers_at_the_ends_of_the_range():
    """A block of any size, with infinities and NaN, of zeros: as the formula on the CPU has it, in the form for the plain products (63 columns) too."""
    for H in (64, 63):
        x = torch.zeros(12, 8, device="cuda", dtype=BF)
        x[:, 0] = torch.tensor([0, 1, 2.0**-60, 2.0**60, 2.0**-110, 2.0**126, -(2.0**126), math.inf, math.nan, 3, -0.0, 2.0**-20], device="cuda").to(BF)
        w1 = torch.zeros(H, 8, device="cuda", dtype=BF)
        w1[:, 0] = _randn(H, gen=_gen(3)).clamp(-3.5, 3.5)
        _, ab, scales = ops.gated_mm(x, w1, w1, 0, 11)
        want = FFN._quantize((x[:, :1].float() * w1[:, 0].float()).unsqueeze(1).expand(12, 2, H), 11)
        rows = [0, 1, 2, 3, 4, 5, 6, 9, 10, 11]
        assert torch.equal(ab[rows], want[0][rows]) and torch.equal(scales, want[1]) and bool((scales[7:9] == 255).all())
        dab, h = ops.gated_dgrad(x, torch.ones(8, H, device="cuda", dtype=BF), ab, scales, 0)
        assert dab[7:9].isnan().all() and h[7:9].isnan().all()


@pytest.mark.parametrize("M,D,H,dtype", [(64, 64, 64, BF), (300, 72, 1000, BF), (999, 2048, 1408, BF), (2100, 256, 5632, BF), (40, 36, 100, BF), (40, 36, 100, F32), (7, 64, 64, F32)])
def test_gradients_of_both_projections_are_tensors_of_their_own(M, D, H, dtype):
    g = _gen(H)
    x, dab = _randn(M, D, gen=g, dtype=dtype), _randn(M, 2, H, gen=g, dtype=dtype)
    for to in (BF, F32) if dtype == BF else (F32,):
        both = ops.gated_wgrad(dab, x, to)
        for i, t in enumerate(both):
            assert t.is_contiguous() and t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size()
            want = dab[:, i].double().t() @ x.double()
            size = dab[:, i].double().abs().t() @ x.double().abs()
            assert bool(((t.double() - want).abs() <= HALF_STEP[to] * want.abs() + M * 2.0**-24 * size).all())
        assert both[0].untyped_storage().data_ptr() != both[1].untyped_storage().data_ptr()
    if dtype == F32:
        return
    x, w1, w3, w2 = (t.requires_grad_() for t in (x, _randn(H, D, gen=g), _randn(H, D, gen=g), _randn(64, H, gen=g)))
    K.gated_ffn(x, w1, w3, w2).float().sum().backward()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    nbytes = w3.grad.numel() * w3.grad.element_size()
    w3.grad = None
    assert before - torch.cuda.memory_allocated() >= nbytes


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("D", [1001, 2048, 16384, 32768])
@pytest.mark.parametrize("size,eps", [(1e-14, 1e-32), (1e-12, 1e-5), (1.0, 1e-5), (1e14, 1e-5), (1e16, 1e-5)])
def test_gradients_of_rows_of_unusual_size(size, eps, D, both, dtype):
    """The norm of rows of any size has a gradient, down to where the square of 1 / rms is no number any more."""
    g = _gen(D)
    x, r = (_randn(19, D, gen=g, dtype=dtype, scale=size) for _ in range(2))
    dy, dh = (_randn(19, D, gen=g, dtype=dtype, scale=s) for s in (1.0, 1 / size))
    w = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dtype)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, h = K.add_rms_norm(*leaves, eps)
    got = torch.autograd.grad((y, h), leaves, (dy, dh)) if both else torch.autograd.grad(y, leaves, dy)
    _check_norm_gradients(got, _norm_gradients(h.detach(), w.detach(), dy, dh if both else None, eps), dtype, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 2048, 16384])
@pytest.mark.parametrize("size,eps", [(1e-14, 1e-32), (1.0, 1e-5), (1e14, 1e-5), (1e16, 1e-5)])
def test_plain_norm_gradients_of_rows_of_unusual_size(size, eps, D, dtype):
    g = _gen(D)
    x, dy = _randn(19, D, gen=g, dtype=dtype, scale=size), _randn(19, D, gen=g, dtype=dtype)
    w = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dtype)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    got = torch.autograd.grad(ops.rms_norm(x, w, eps)[0], leaves, dy)
    _check_norm_gradients(got, _norm_gradients(x.detach(), w.detach(), dy, None, eps), dtype, dtype)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_fp32_activation_relative_to_the_value(act):
    """fp32 operands: the activation and its derivative to a few roundings of the value, far out on the negative side too."""
    a = torch.linspace(-60 if act == "silu" else -9.9, 10, 4001, device="cuda").unsqueeze(1)
    one = torch.ones(1, 1, device="cuda")
    # (in forms that keep their digits: 1 + erf and 1 + tanh are zero in 64 bits from -8.3 and 2 u = -37 on)
    d = a.double().requires_grad_()
    s = {"silu": lambda t: torch.sigmoid(t), "gelu": lambda t: 0.5 * torch.erfc(-t * 0.5**0.5),
         "gelu_tanh": lambda t: torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (t + 0.044715 * t**3))}[act](d)
    v = d * s
    (dv,) = torch.autograd.grad(v.sum(), d)
    s, v, d = s.detach(), v.detach(), d.detach()
    # The argument of the exponential is off by a few of its own roundings, which is that much of the value: none for silu, |u| for gelu_tanh, a^2 / 2 and the
    # constant in erfc's argument for gelu.  Functions: erfc to 4 units in the last place (2^-23 each), exp to 2, sums and products to a half.
    u = {"silu": 0 * d, "gelu": d.square(), "gelu_tanh": 1.5957691216 * d * (1 + 0.044715 * d * d)}[act].abs()
    tol = (16 + 5 * u) * 2.0**-24
    h, ab, _ = ops.gated_mm(a, one, one, FFN.ACTS[act], 16)
    assert torch.equal(ab[:, 0], a)
    assert bool(((h.double() - v * d).abs() <= (tol + 2.0**-24) * (v * d).abs()).all()), float(((h.double() - v * d).abs() / (v * d).abs().clamp_min(1e-300)).max())
    ab = torch.stack((a, torch.ones_like(a)), 1)
    dab, h = ops.gated_dgrad(torch.ones_like(a), one, ab, torch.empty(0, dtype=torch.uint8, device="cuda"), FFN.ACTS[act])
    assert bool(((h.double() - v).abs() <= tol * v.abs()).all()) and torch.equal(dab[:, 1], h)
    # the derivative is a sum that cancels: relative to its terms, both of which carry the same exponential
    terms = s + (dv - s).abs()
    assert bool(((dab[:, 0].double() - dv).abs() <= (tol + 8 * 2.0**-24) * terms).all()), float(((dab[:, 0].double() - dv).abs() / terms).max())


@pytest.mark.parametrize("form,both", [("norm", True), ("norm", False), ("fp8", True), ("fp8", False), ("fp8 of x alone", False)])
@pytest.mark.parametrize("D", [64, 1001, 4096, 32768])
def test_gradient_of_an_fp32_weight_beside_bf16_operands(D, form, both):
    """It is summed in fp32 and not rounded to the operands' type."""
    g = _gen(D)
    x, r, dy, dh = (_randn(300, D, gen=g) for _ in range(4))
    w = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
    alone = form == "fp8 of x alone"
    leaves = [t.requires_grad_() for t in ((x, w) if alone else (x, r, w))]
    out = K.add_rms_norm(*leaves) if form == "norm" else K.add_rms_norm_fp8(x, None if alone else r, w)
    got = torch.autograd.grad(out[:2], leaves, (dy, dh)) if both else torch.autograd.grad(out[0], leaves, dy)
    # (the weight itself is taken in the operands' type, as ``rms_norm`` takes it)
    _check_norm_gradients(got, _norm_gradients(x.detach() if alone else out[1].detach(), w.detach().to(BF), dy, dh if both else None, 1e-5), BF, F32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [200, 1001, 4096, 32768])
@pytest.mark.parametrize("size,weight,eps", [(2.0**-55, 2.0**-65, 2e-38), (2.0**-55, 2.0**-80, 2e-38), (2.0**50, 2.0**80, 1e-5), (2.0**-20, 2.0**-100, 1e-30), (1.0, 2.0**-120, 1e-5)])
def test_8_bit_norm_of_products_outside_of_the_range(D, size, weight, eps, dtype):
    """h w or 448 / max |h w| are no fp32 numbers, the norm and its scale are."""
    g = _gen(D)
    x = _randn(9, D, gen=g, dtype=dtype, scale=size)
    x[4] = 0
    w = (weight * (1 + 0.1 * torch.randn(D, device="cuda", generator=g))).to(dtype)
    for keep in (False, True):
        y, h, q, scale = K.add_rms_norm_fp8(x, None, w, eps, keep)
        yd = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps) * w.double()
        top = yd.abs().amax(-1, keepdim=True)
        want = torch.where(top < 2.0**-100, 1.0, top / 448)
        assert bool(((scale.double() - want).abs() <= ARITHMETIC * want).all())
        err = (q.double() * scale.double() - yd).abs()
        assert bool((err <= (1 + 2.0**-14) * torch.maximum(yd.abs() * 2.0**-4, scale.double() * 2.0**-10)).all())
        if keep:
            assert torch.equal(y, K.add_rms_norm(x, torch.zeros_like(x), w, eps)[0])
