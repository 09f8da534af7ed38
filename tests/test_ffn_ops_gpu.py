"""The feed-forward block's kernels against the formulas in 64 bits.

Tolerances are relative to the size of the result (its root mean square over the tensor, or the value where that is larger).  A rounding to bf16 is off by at
most 2^-8 of the value, a sum of n products in fp32 by at most n 2^-24 of the sum of the magnitudes and by about sqrt(n) 2^-24 of it; what a formula rounds on its
way (h, da, db, and the codes of a, b) adds its own half step, spread over a sum of n terms like noise: the factors below count those."""
import math

import pytest
import torch
import torch.nn.functional as F

import autoparallel_b200.ops as K
from autoparallel_b200.ops import ffn_ops as FFN
from autoparallel_b200.ops.library import ops, reference_impls

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
ACTS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}
HALF_STEP = {BF: 2.0**-8, F32: 2.0**-24}


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


def _close(got, want, tol):
    want = want.double()
    size = torch.maximum(want.abs(), want.square().mean().sqrt()) if want.numel() else want
    err = (got.double() - want).abs()
    assert got.shape == want.shape and bool((err <= tol * size + 1e-30).all()), float((err / size.clamp_min(1e-30)).max())


def _held(x):
    """What 8 bits hold of x, in 64 bits."""
    k = x.shape[-1]
    b = F.pad(x.double(), (0, -k % 32)).unflatten(-1, (-1, 32))
    e = (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 1).clamp_min(-120).double()
    return (torch.clamp(torch.round(b / torch.exp2(e - 6)), -127, 127) * torch.exp2(e - 6)).flatten(-2)[..., :k]


def _kept(ab, scales):
    """The values of what was kept of both projections, in 64 bits."""
    if ab.is_floating_point():
        return ab.double()
    unit = torch.exp2(scales.double() - 127 - (6 if ab.dtype is torch.int8 else 14)).masked_fill(scales == 255, float("nan"))
    return ab.double() * unit.repeat_interleave(32, -1)[..., : ab.shape[-1]]


def _tops(v):
    """The largest magnitude of every value's block of 32."""
    k = v.shape[-1]
    return F.pad(v, (0, -k % 32)).unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(*v.shape[:-1], -1, 32).flatten(-2)[..., :k]


# ------------------------------------------------------------------------------------ 8-bit checkpoints
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 3, 64), (7, 1000), (64, 4096), (129, 257), (0, 64), (4, 0), (9,), (1023, 96)])
def test_mx8(shape, dtype):
    x = _randn(*shape, gen=_gen(1), dtype=dtype, scale=5.0)
    if x.numel() > 40:
        x.view(-1)[3] = float("inf")
        x.view(-1)[40] = float("nan")
        x.view(-1)[-1] = -0.0
    codes, scales = K.mx8_quantize(x)
    want = reference_impls["mx8_quantize"](x.cpu())
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    for t in (BF, F32):
        got = K.mx8_dequantize(codes, scales, t).cpu()
        ref = reference_impls["mx8_dequantize"](*want, t)
        assert got.dtype == t and torch.equal(got.nan_to_num(nan=-1.0), ref.nan_to_num(nan=-1.0))


def test_mx8_extremes():
    x = torch.zeros(9, 32, device="cuda")
    x[1, 0], x[1, 1] = torch.finfo(F32).max, -torch.finfo(F32).max
    x[2, 0], x[3, 0], x[4, 3] = 2.0**-126, 2.0**-149, float("inf")
    x[5, 4], x[6] = float("nan"), 127.6
    x[7] = torch.arange(32, device="cuda") / 32.0 * 2.0**-125
    x[8, 5] = -127.5
    codes, scales = K.mx8_quantize(x)
    want = reference_impls["mx8_quantize"](x.cpu())
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])


@pytest.mark.parametrize("k", [1, 31, 223, 225, 231, 449, 457, 900, 1003])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_mx8_of_rows_that_begin_anywhere(k, dtype):
    """Every way for a row to begin, blocks of very different sizes, of zeros, at the clamp, and with values that are not numbers."""
    g = _gen(k)
    x = _randn(37, k, gen=g, dtype=F32) * torch.exp2(torch.randint(-90, 90, (37, k), device="cuda", generator=g).float().div(16).floor().mul(16))
    draw = torch.rand(37, k, device="cuda", generator=g)
    x = torch.where(draw < 0.01, 0.0, torch.where(draw < 0.02, 255.75 / 256 * torch.exp2(torch.log2(x.abs()).ceil()), x))
    x[3::7] = 0.0
    for i, v in enumerate((math.nan, math.inf, -math.inf, 3e38, -1e-40)):
        x[5 * i + 2, (i * 97) % k] = v
    x = x.to(dtype)
    codes, scales = K.mx8_quantize(x)
    want = K.mx8_quantize(x.cpu())
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    for to in (BF, F32):
        a, b = K.mx8_dequantize(codes, scales, to).cpu(), K.mx8_dequantize(*want, to)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_mx8_of_strided_and_shifted_operands():
    base = _randn(65, 130, gen=_gen(2), dtype=F32)
    for x in (base.t(), base[:, 1:], base[1:, 2:66], base[::2], base.flatten()[3:].view(-1)[:8192].view(64, 128)):
        codes, scales = K.mx8_quantize(x)
        want = reference_impls["mx8_quantize"](x.cpu())
        assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
        assert torch.equal(K.mx8_dequantize(codes[1:], scales[1:]).cpu(), reference_impls["mx8_dequantize"](want[0][1:], want[1][1:], BF))


# ------------------------------------------------------------------------------------ norm
NORM_SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 3, 256), (9, 264), (17, 1000), (33, 1001), (4, 1024), (5, 2048), (3, 4096), (2, 8191), (3, 8192), (2, 16384),
               (1, 32768), (2, 32767), (1500, 512), (700, 1040), (64,), (0, 64)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_add_rms_norm(shape, dtype):
    g = _gen(4)
    x, r, dy, dh = (_randn(*shape, gen=g, dtype=dtype) for _ in range(4))
    w = (1 + 0.1 * torch.randn(shape[-1], device="cuda", generator=g)).to(dtype)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = K.add_rms_norm(*leaves, 1e-5)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    if shape[-1] % 8 == 0:
        assert torch.equal(y, ops.rms_norm(h, w, 1e-5)[0])
    hd, wd = h.detach().double().requires_grad_(), w.double().requires_grad_()
    yd = hd * torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * wd
    # one rounding; 1 / rms by an instruction of 2^-22, sums of D squares in chains of D / threads and a tree
    arithmetic = 16 * 2.0**-22
    _close(y, yd.detach(), HALF_STEP[dtype] + arithmetic)
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    if not x.numel():
        assert got[0].shape == x.shape and not got[2].any()
        return
    dx, dw = torch.autograd.grad((yd, hd * 1), (hd, wd), (dy.double(), dh.double()))
    _close(got[0], dx, HALF_STEP[dtype] + arithmetic)
    assert torch.equal(got[0], got[1])
    _close(got[2], dw, HALF_STEP[dtype] + arithmetic + math.sqrt(x.numel() / shape[-1]) * 2.0**-23)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_add_rms_norm_with_an_fp32_weight(dtype):
    x, r = (_randn(6, 128, gen=_gen(s), dtype=dtype).requires_grad_() for s in (1, 2))
    w = torch.randn(128, device="cuda").requires_grad_()
    y, h = K.add_rms_norm(x, r, w)
    assert torch.equal(y, ops.rms_norm(h, w, 1e-5)[0])
    gw = torch.autograd.grad(y.float().sum(), w)[0]
    assert gw.dtype == F32 and gw.shape == w.shape


def test_add_rms_norm_of_rows_that_are_not_numbers():
    """A row with an infinity or a NaN spoils no other row, and comes out as the formula has it."""
    x, r = (_randn(6, 512, gen=_gen(s)) for s in (1, 2))
    clean = K.add_rms_norm(x, r, torch.ones(512, device="cuda", dtype=BF))
    clean8 = K.add_rms_norm_fp8(x, r, torch.ones(512, device="cuda", dtype=BF))
    x[1, 7], x[3, 9], x[4], r[4] = float("inf"), float("nan"), 0, 0
    w = torch.ones(512, device="cuda", dtype=BF)
    y, h = K.add_rms_norm(x, r, w)
    q8 = K.add_rms_norm_fp8(x, r, w)
    for row in (0, 2, 5):
        assert torch.equal(y[row], clean[0][row]) and torch.equal(q8[2][row].float(), clean8[2][row].float()) and torch.equal(q8[3][row], clean8[3][row])
    assert y[1, 7].isnan() and not y[1, :7].any() and y[3].isnan().all() and not y[4].any()
    assert q8[3][3].isnan() and q8[3][1].isnan() and q8[3][4].item() == 1.0 and not q8[2][4].float().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 64), (2, 3, 256), (17, 1000), (33, 1001), (3, 4096), (2, 8191), (2, 16384), (1, 32768), (64,), (0, 64)])
def test_add_rms_norm_fp8(shape, residual, keep, dtype):
    g = _gen(6)
    x = _randn(*shape, gen=g, dtype=dtype)
    r = _randn(*shape, gen=g, dtype=dtype) if residual else None
    w = (1 + 0.1 * torch.randn(shape[-1], device="cuda", generator=g)).to(dtype)
    y, h, q, scale = K.add_rms_norm_fp8(x, r, w, keep=keep)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (*shape[:-1], 1)
    if residual:
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
    else:
        assert h is x
    if keep:
        assert torch.equal(y, K.add_rms_norm(x, r if residual else torch.zeros_like(x), w)[0])
    else:
        assert y is None
    if not x.numel():
        return
    yd = h.double() * torch.rsqrt(h.double().pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    top = yd.abs().amax(-1, keepdim=True)
    assert bool(((scale.double() - top / 448).abs() <= 16 * 2.0**-22 * top / 448).all())
    # e4m3: half a step is 2^-4 of the value, 2^-10 below the normal range, in units of the scale
    err = (q.double() * scale.double() - yd).abs()
    assert bool((err <= (1 + 2.0**-14) * torch.maximum(yd.abs() * 2.0**-4, scale.double() * 2.0**-10)).all())


def test_add_rms_norm_fp8_gradients():
    g = _gen(8)
    x, r, dy, dh = (_randn(37, 512, gen=g) for _ in range(4))
    w = _randn(512, gen=g)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h, q, scale = K.add_rms_norm_fp8(*leaves)
    assert not q.requires_grad and not scale.requires_grad
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    other = [t.clone().requires_grad_() for t in (x, r, w)]
    want = torch.autograd.grad(K.add_rms_norm(*other), other, (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    y, h, q, scale = K.add_rms_norm_fp8(leaves[0], None, leaves[1])
    got = torch.autograd.grad(y, leaves, dy)
    other = [t.clone().requires_grad_() for t in (x, w)]
    want = torch.autograd.grad(ops.rms_norm(*other, 1e-5)[0], other, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_where_one_result_is_used():
    x, r = (_randn(9, 264, gen=_gen(s)).requires_grad_() for s in (1, 2))
    w = torch.ones(264, device="cuda", dtype=BF, requires_grad=True)
    gx, gr, gw = torch.autograd.grad(K.add_rms_norm(x, r, w)[1].sum(), (x, r, w))
    assert bool((gx == 1).all()) and bool((gr == 1).all()) and not gw.any()
    dy = _randn(9, 264, gen=_gen(3))
    got = torch.autograd.grad(K.add_rms_norm(x, r, w)[0], (x, r, w), dy)
    h = (x + r).detach().requires_grad_()
    want = torch.autograd.grad(ops.rms_norm(h, w, 1e-5)[0], (h, w), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[1])


def test_gradients_do_not_share_memory():
    """Where only the sum is used its gradient is passed on; what becomes of one leaf's gradient is not seen in another's, nor in the caller's."""
    w = torch.ones(264, device="cuda", dtype=BF)
    for used, f in ((0, lambda *a: K.add_rms_norm(*a)[1]), (1, lambda *a: K.add_rms_norm_fp8(*a)[1]), (2, lambda *a: sum(K.add_rms_norm(*a)))):
        x, r = (_randn(9, 264, gen=_gen(s)).requires_grad_() for s in (1, 2))
        dy = torch.ones_like(x)
        f(x, r, w).backward(dy)
        assert len({t.data_ptr() for t in (dy, x.grad, r.grad)}) == 3, used
        x.grad.zero_()
        assert bool((dy == 1).all()) and (used == 2 or bool((r.grad == 1).all())), used
        r.grad.zero_()
        assert bool((dy == 1).all()), used


# ------------------------------------------------------------------------------------ gated block
def _gated(M, D, H, N, dtype=BF, seed=0):
    g = _gen(seed)
    x = _randn(M, D, gen=g, dtype=dtype)
    w1, w3 = (_randn(H, D, gen=g, dtype=dtype, scale=max(D, 1) ** -0.5) for _ in range(2))
    return x, w1, w3, _randn(N, H, gen=g, dtype=dtype, scale=max(H, 1) ** -0.5), _randn(M, N, gen=g, dtype=dtype)


def _products(x, w1, w3):
    return x.double() @ w1.double().t(), x.double() @ w3.double().t()


# rows: few-row kernel, split kernel, single CTAs, pairs, wide pairs; columns: parts of tiles and of blocks of 32
FORMS = [(1, 64, 8), (1, 4096, 1024), (3, 256, 40), (8, 512, 264), (16, 256, 96), (17, 2048, 1408), (32, 128, 72), (33, 64, 136), (100, 320, 200), (128, 8, 64), (130, 1288, 520),
         (200, 2048, 4096), (256, 64, 128), (300, 136, 2056), (513, 256, 1416), (999, 2048, 1408), (1024, 512, 5632), (2100, 72, 1000), (4096, 4416, 1032)]


@pytest.mark.parametrize("bits", [0, 8, 16])
@pytest.mark.parametrize("M,D,H", FORMS)
def test_gated_mm(M, D, H, bits):
    act = sorted(ACTS)[(M + D + H) % 3]
    x, w1, w3, _, _ = _gated(M, D, H, 8, seed=M)
    h, ab, scales = ops.gated_mm(x, w1, w3, FFN.ACTS[act], bits)
    a, b = _products(x, w1, w3)
    acc = 4 * math.sqrt(D) * 2.0**-24  # of the products' size
    _close(h, ACTS[act](a) * b, HALF_STEP[BF] + 8 * acc)
    if bits:
        exact = torch.stack((a, b), 1)
        assert ab.dtype == (torch.int8 if bits == 8 else torch.int16) and scales.shape == (M, 2, -(-H // 32))
        got = _kept(ab, scales)
        # half a step of the block's codes, a whole one at the block's top, which rounds to 2^(bits - 1) and is held as one less; a top at a power of two may
        # fall on either side of it
        step = torch.exp2(torch.floor(torch.log2(_tops(exact) * (1 + 2.0**-15))) - (bits - 2))
        near = exact.abs() > (2 ** (bits - 1) - 0.6 - 2.0**-14 * 2 ** (bits - 1)) * step
        # and the product's own error, which is of the size of the terms and not of a value that they cancel to: the accumulator is rounded D / 16
        # times at its running size, about the root mean square of the results, D / 16 2^-24 <= 4 sqrt(D) 2^-24 for D <= 4096 and 1.04 of it for 4416
        size = torch.maximum(exact.abs(), 1.04 * exact.square().mean().sqrt())
        assert bool(((got - exact).abs() <= torch.where(near, 1.0, 0.5) * step + 1e-4 * step + acc * size).all())
        assert bool((scales.int() >= bits - 1).all())
    else:
        assert ab.numel() == 0 and scales.numel() == 0


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("M,N,H", FORMS)
def test_gated_dgrad(M, N, H, bits):
    act = sorted(ACTS)[(M + N + H) % 3]
    x, w1, w3, w2, dy = _gated(M, 64, H, N, seed=M + 1)
    _, ab, scales = ops.gated_mm(x, w1, w3, FFN.ACTS[act], bits)
    dab, h = ops.gated_dgrad(dy, w2, ab, scales, FFN.ACTS[act])
    a, b = (t.clone().requires_grad_() for t in _kept(ab, scales).unbind(1))
    hd = ACTS[act](a) * b
    da, db = torch.autograd.grad(hd, (a, b), dy.double() @ w2.double())
    tol = HALF_STEP[BF] + 32 * math.sqrt(N) * 2.0**-24
    _close(dab[:, 0], da, tol)
    _close(dab[:, 1], db, tol)
    _close(h, hd.detach(), HALF_STEP[BF] + 2.0**-18)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("M,H", [(5, 64), (5, 63), (300, 2056)])
def test_gated_dgrad_of_values_near_the_largest(M, H, bits):
    """The codes' values are exact up to the end of fp32's range."""
    g = _gen(M + H)
    a, b = (_randn(M, H, gen=g, dtype=F32, scale=s).clamp(-2e38, 2e38) for s in (1.0, 1e38))
    w2, dy = _randn(64, H, gen=g, scale=0.125), _randn(M, 64, gen=g, scale=1e-33)
    ab, scales = FFN._quantize(torch.stack((a, b), 1), bits)
    dab, h = ops.gated_dgrad(dy, w2, ab, scales, 0)
    a, b = (t.clone().requires_grad_() for t in _kept(ab, scales).unbind(1))
    hd = F.silu(a) * b
    da, db = torch.autograd.grad(hd, (a, b), dy.double() @ w2.double())
    tol = HALF_STEP[BF] + 32 * math.sqrt(64) * 2.0**-24
    _close(dab[:, 0], da, tol)
    _close(dab[:, 1].double() * 2.0**110, db * 2.0**110, tol)  # (away from the 1e-30 of _close)
    # silu(a) b passes the largest bf16 number, 3.39e38, for some: with |b| <= 2e38 wherever silu(a) > 1.7.  Those are infinities; next to it either is right.
    hd, top = hd.detach(), torch.finfo(BF).max
    over, below = hd.abs() > top * (1 + 2.0**-8), hd.abs() < top * (1 - 2.0**-8)
    assert torch.equal(h[over].double(), math.inf * hd[over].sign())
    _close(torch.where(below, h, 0), torch.where(below, hd, 0), HALF_STEP[BF] + 2.0**-18)


@pytest.mark.parametrize("M,D,H", FORMS)
def test_gated_dx_and_wgrad(M, D, H):
    x, w1, w3, _, _ = _gated(M, D, H, 8, seed=M + 2)
    dab = _randn(M, 2, H, gen=_gen(M))
    dx = ops.gated_dx(dab, w1, w3)
    da, db = dab.double().unbind(1)
    _close(dx, da @ w1.double() + db @ w3.double(), HALF_STEP[BF] + 8 * math.sqrt(2 * H) * 2.0**-24)
    dw1, dw3 = ops.gated_wgrad(dab, x, BF)
    _close(dw1, da.t() @ x.double(), HALF_STEP[BF] + 8 * math.sqrt(M) * 2.0**-24)
    _close(dw3, db.t() @ x.double(), HALF_STEP[BF] + 8 * math.sqrt(M) * 2.0**-24)
    w32 = ops.gated_wgrad(dab, x, F32)
    _close(w32[1], db.t() @ x.double(), 16 * math.sqrt(M) * 2.0**-24 + 2.0**-20)


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
@pytest.mark.parametrize("M,D,H,N,dtype", [(1, 64, 96, 64, BF), (40, 128, 264, 72, BF), (300, 256, 520, 256, BF), (1030, 512, 1408, 512, BF), (7, 20, 33, 12, BF),
                                           (65, 36, 100, 20, BF), (50, 128, 96, 128, F32), (9, 13, 21, 5, F32)])
def test_gated_ffn_training(M, D, H, N, dtype, checkpoint):
    for act in sorted(ACTS):
        x, w1, w3, w2, dy = _gated(M, D, H, N, dtype, seed=M + 3)
        leaves = [t.requires_grad_() for t in (x, w1, w3, w2)]
        y = K.gated_ffn(*leaves, act=act, checkpoint=checkpoint)
        got = torch.autograd.grad(y, leaves, dy)
        d = [t.detach().double() for t in leaves]
        a, b = _products(d[0], d[1], d[2])
        # forward: h rounded, then the result; backward: a, b, da, db, h and the result rounded (fp32: the products' own rounding of sums)
        step = HALF_STEP[dtype] if dtype == BF else 64 * 2.0**-24
        _close(y, (ACTS[act](a) * b) @ d[3].t(), 3 * step)
        xk = d[0]
        if checkpoint == "mx8":
            xk = _held(d[0])
            _, ab, scales = ops.gated_mm(*leaves[:3], FFN.ACTS[act], 8)
            a, b = K.mx8_dequantize(ab, scales, F32).double().unbind(1)
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        h = ACTS[act](a) * b
        da, db = torch.autograd.grad(h, (a, b), dy.double() @ d[3])
        want = (da @ d[1] + db @ d[2], da.t() @ xk, db.t() @ xk, dy.double().t() @ h.detach())
        if dtype == F32:
            for u, v in zip(got, want):
                _close(u, v, 5 * step)
            continue
        # What each rounding can do to a term, in magnitudes: a and b are off by 2^-15 of their block's top ("full": 16-bit codes; the 8-bit ones are known
        # here), da, db and h by a half step of theirs; |act'| <= 1.13 and |act''| <= 0.8 for all three.  The bound of a sum is the sum of the bounds (1.02:
        # products of two errors, and twice 2^-15 at a block's top), then the result's own rounding and 2^-16 for the fp32 sums.
        e, dh = HALF_STEP[BF], (dy.double() @ d[3]).abs()
        av, bv, hv = a.detach().abs(), b.detach().abs(), h.detach().abs()
        ka, kb = ((2.0**-14 * _tops(t) if checkpoint == "full" else torch.zeros_like(t)) for t in (av, bv))
        off_a = e * da.abs() + dh * (0.8 * ka * bv + 1.13 * kb)
        off_b = e * db.abs() + dh * 1.13 * ka
        off_h = e * hv + 1.13 * ka * bv + ACTS[act](a.detach()).abs() * kb
        w1a, w3a, xa, dya = d[1].abs(), d[2].abs(), xk.abs(), dy.double().abs()
        for u, v, off in zip(got, want, (off_a @ w1a + off_b @ w3a, off_a.t() @ xa, off_b.t() @ xa, dya.t() @ off_h)):
            assert bool(((u.double() - v).abs() <= 1.02 * off + e * v.abs() + 2.0**-16 * v.square().mean().sqrt()).all())
            # and as noise: a rounding's error is at most a half step, spread evenly, sqrt(1/3) of it; two of them on the way of a result, and the codes'
            assert u.numel() < 1000 or float((u.double() - v).norm() / v.norm()) <= math.sqrt(3 / 3) * e


def test_gated_ffn_leading_dims_strides_and_partial_gradients():
    g = _gen(21)
    x = _randn(3, 70, 128, gen=g)
    w1, w3, w2 = _randn(264, 128, gen=g, scale=0.1), _randn(264, 128, gen=g, scale=0.1), _randn(96, 264, gen=g, scale=0.1)
    y = K.gated_ffn(x, w1, w3, w2)
    assert y.shape == (3, 70, 96)
    for args in ((x.transpose(0, 1).contiguous().transpose(0, 1), w1, w3, w2), (x, w1.t().contiguous().t(), w3, w2.t().contiguous().t()),
                 (F.pad(x, (0, 3))[..., :128], F.pad(w1, (8, 8))[:, 8:136], F.pad(w3, (1, 0))[:, 1:], w2)):
        assert torch.equal(K.gated_ffn(*args), y)
    dy = _randn(3, 70, 96, gen=g)
    for checkpoint in ("full", "mx8"):
        every = [t.clone().requires_grad_() for t in (x, w1, w3, w2)]
        want = torch.autograd.grad(K.gated_ffn(*every, checkpoint=checkpoint), every, dy)
        for i in range(4):
            some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w1, w3, w2))]
            (got,) = torch.autograd.grad(K.gated_ffn(*some, checkpoint=checkpoint), some[i], dy)
            assert torch.equal(got, want[i]), i
        # a gradient that is not dense: of a sum, of a transposed result
        a, b = (torch.autograd.grad(f(K.gated_ffn(*every, checkpoint=checkpoint)), every[0])[0]
                for f in (lambda t: t.float().sum(), lambda t: (t * torch.ones_like(t)).float().sum()))
        assert torch.equal(a, b)


@pytest.mark.parametrize("M", [5, 33, 300])
@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_gated_ffn_of_rows_that_lie_on_one_another(M, checkpoint):
    """An expanded x, expanded weights, and the expanded gradient that a sum over rows has: the results of the same values written out."""
    x, w1, w3, w2, dy = _gated(M, 128, 264, 96)
    x, w1, w3, w2, dy = x[:1].expand(M, 128), w1[:1].expand(264, 128), w3, w2[:1].expand(96, 264), dy[:1].expand(M, 96)
    out = []
    for f in (lambda t: t, lambda t: t.contiguous()):
        leaves = [f(t.detach()).requires_grad_() for t in (x, w1, w3, w2)]
        y = K.gated_ffn(*leaves, checkpoint=checkpoint)
        out.append((y, *torch.autograd.grad(y, leaves, f(dy))))
        out[-1] += (*torch.autograd.grad(K.gated_ffn(*leaves, checkpoint=checkpoint).sum(0), leaves, dy[0]),)
    for i, (a, b) in enumerate(zip(*out)):
        assert torch.equal(a, b), i
    three = x.unsqueeze(0).expand(3, M, 128)
    assert torch.equal(K.gated_ffn(three, w1, w3, w2), K.gated_ffn(three.contiguous(), w1, w3, w2))


def test_gated_ffn_where_values_are_not_numbers():
    """A row that holds a NaN or an infinity spoils no other row, in either direction."""
    x, w1, w3, w2, dy = _gated(300, 64, 264, 64, seed=5)
    for checkpoint in ("full", "mx8"):
        outs = []
        for bad in (False, True):
            xb = x.clone()
            if bad:
                xb[7, 3], xb[290, 0] = float("nan"), float("inf")
            xb.requires_grad_()
            y = K.gated_ffn(xb, w1, w3, w2.clone().requires_grad_(), checkpoint=checkpoint)
            outs.append((y.detach(), torch.autograd.grad(y, xb, dy)[0]))
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[7] = keep[290] = False
        for a, b in zip(*outs):
            assert torch.equal(a[keep], b[keep]) and b[7].isnan().all()


def test_gated_block_of_nothing():
    for dtype in (BF, F32):
        for m, d, h, n in ((0, 8, 16, 8), (3, 0, 16, 8), (3, 8, 0, 8), (3, 8, 16, 0)):
            x, w1, w3, w2 = (torch.randn(*s, device="cuda").to(dtype).requires_grad_() for s in ((m, d), (h, d), (h, d), (n, h)))
            for checkpoint in ("full", "mx8"):
                y = K.gated_ffn(x, w1, w3, w2, checkpoint=checkpoint)
                assert y.shape == (m, n) and not y.any()
                for t, g in zip((x, w1, w3, w2), torch.autograd.grad(y.sum(), (x, w1, w3, w2))):
                    assert g.shape == t.shape and not g.any()


# ------------------------------------------------------------------------------------ together, repeated, captured, on other streams
def _block(x, delta, norm, w1, w3, w2, checkpoint):
    n, h = K.add_rms_norm(delta, x, norm)
    return h + K.gated_ffn(n, w1, w3, w2, checkpoint=checkpoint)


def _block_leaves(M=300, D=256, H=520, seed=30):
    g = _gen(seed)
    x, delta = _randn(M, D, gen=g), _randn(M, D, gen=g)
    norm = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(BF)
    return [t.requires_grad_() for t in (x, delta, norm, *(_randn(*s, gen=g, scale=s[1] ** -0.5) for s in ((H, D), (H, D), (D, H))))], _randn(M, D, gen=g)


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_half_a_layer_against_separate_operators(checkpoint):
    """Norm, block and residual together: as near to 64 bits as the operators that the framework had."""
    leaves, dy = _block_leaves()
    got = torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy)
    x, delta, norm, w1, w3, w2 = leaves
    h = x + delta
    n = K.rms_norm(h, norm)
    y = h + ops.mm_nd(K.swiglu(ops.mm_nd(n, w1, True, BF), ops.mm_nd(n, w3, True, BF)), w2, True, BF)
    unfused = torch.autograd.grad(y, leaves, dy)
    d = [t.detach().double().requires_grad_() for t in leaves]
    hd = d[0] + d[1]
    nd = hd * torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * d[2]
    yd = hd + (F.silu(nd @ d[3].t()) * (nd @ d[4].t())) @ d[5].t()
    want = torch.autograd.grad(yd, d, dy.double())
    for a, b, c in zip(got, unfused, want):
        err, before = ((t.double() - c).norm() / c.norm() for t in (a, b))
        # 8 bits hold a value to 2^-7 of its block's largest; x, a and b are rounded so
        assert err <= (1.5 * before + 1e-6 if checkpoint == "full" else 2.0**-6), (float(err), float(before))


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_the_same_bits_every_time_and_on_other_streams(checkpoint):
    leaves, dy = _block_leaves()
    first = torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i in range(6):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, first))


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_captured_and_replayed(checkpoint):
    """Two graphs of the same calls, replayed in turn on new inputs, give what separate calls give."""
    leaves, dy = _block_leaves(M=130)
    x = leaves[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy))
        graphs.append(g)
    for seed in (1, 2):
        with torch.no_grad():
            x.copy_(_randn(*x.shape, gen=_gen(seed)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(_block(*leaves, checkpoint), leaves, dy)
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))
    for g in graphs:
        g.reset()


def test_decoding_in_a_graph():
    leaves, _ = _block_leaves(M=1, D=512, H=1408)
    with torch.no_grad():
        want = _block(*leaves, "full")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _block(*leaves, "full")
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        g.reset()


@pytest.mark.parametrize("M,D,H", [(1, 1024, 4096), (8, 2048, 1408), (16, 512, 2816), (20, 512, 1024), (4, 4096, 512)])
@pytest.mark.parametrize("graph", [False, True])
def test_weights_that_are_written_just_before(M, D, H, graph):
    """A few rows: the second product's weights are read while the first product runs, but never before what wrote them has ended."""
    x, w1, w3, w2, _ = _gated(M, D, H, D, seed=5)
    source, one = w2.float(), torch.ones((), device="cuda")
    kept = w2.clone()

    def calls():
        out = []
        for i in range(12):
            one.neg_()
            if i % 2:
                out.append(K.gated_ffn(x, w1, w3, ops.dtype_cast(source * one, BF)))  # (by a kernel of the framework's own)
            else:
                torch.mul(kept, one.to(BF), out=w2)
                out.append(K.gated_ffn(x, w1, w3, w2))
        return out

    want = K.gated_ffn(x, w1, w3, kept)
    torch.cuda.synchronize()
    if graph:
        g = torch.cuda.CUDAGraph()
        calls()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            got = calls()
        for _ in range(3):
            g.replay()
    else:
        got = calls()
    for i, y in enumerate(got):
        assert torch.equal(y, want if i % 2 else -want), i


def test_rows_do_not_depend_on_each_other():
    """A row of a batch is the row by itself where both go to the same kernel, and as near as the products' sums elsewhere."""
    x, w1, w3, w2, _ = _gated(1030, 256, 520, 256, seed=8)
    y = K.gated_ffn(x, w1, w3, w2)
    assert torch.equal(K.gated_ffn(x[:1029], w1, w3, w2), y[:1029])
    _close(K.gated_ffn(x[5:6], w1, w3, w2), y[5:6].double(), 4 * HALF_STEP[BF])


def test_reserved_sms_and_makes_room(loaded):
    ext = loaded.extension()
    x, w1, w3, w2, dy = _gated(1030, 256, 520, 256, seed=9)
    leaves = [t.requires_grad_() for t in (x, w1, w3, w2)]
    want = torch.autograd.grad(K.gated_ffn(*leaves), leaves, dy)
    try:
        ext.gemm_set_reserved_sms(16)
        got = torch.autograd.grad(K.gated_ffn(*leaves), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ext.gemm_set_reserved_sms(0)
        ext.gemm_set_dynamic_tiles(True)
        got = torch.autograd.grad(K.gated_ffn(*leaves), leaves, dy)
    finally:
        ext.gemm_set_reserved_sms(0)
        ext.gemm_set_dynamic_tiles(False)
    for a, b in zip(got, want):
        _close(a, b.double(), 6 * HALF_STEP[BF])


def test_second_derivatives_are_refused():
    x, w1, w3, w2, _ = _gated(8, 64, 64, 64)
    x.requires_grad_()
    (g,) = torch.autograd.grad(K.gated_ffn(x, w1, w3, w2).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        g.float().sum().backward()
    r = torch.ones_like(x).requires_grad_()
    y, h = K.add_rms_norm(x, r, torch.ones(64, device="cuda", dtype=BF))
    (g,) = torch.autograd.grad((y * y + h).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        g.float().sum().backward()
    y = ops.gated_ffn(x, w1, w3, w2, 0, 0)[0]
    with pytest.raises(RuntimeError, match="kept nothing"):
        y.float().sum().backward()


def test_refusals():
    x = torch.randn(4, 8, device="cuda")
    for args in ((x, x.cpu(), x[0]), (x, x, x[0].cpu())):
        with pytest.raises(ValueError, match="different devices"):
            K.add_rms_norm(*args)
    w1, w2 = torch.randn(16, 8, device="cuda"), torch.randn(8, 16, device="cuda")
    with pytest.raises(ValueError, match="different devices"):
        K.gated_ffn(x, w1, w1.cpu(), w2)
    with pytest.raises(RuntimeError, match="act 0 to 2"):
        ops.gated_mm(x, w1, w1, 3, 0)
    with pytest.raises(RuntimeError, match="bits 0, 8 or 16"):
        ops.gated_mm(x, w1, w1, 0, 4)
    _, ab, scales = ops.gated_mm(x, w1, w1, 0, 8)
    with pytest.raises(RuntimeError, match="uint8 scales"):
        ops.gated_dgrad(x, w2, ab, scales[:2], 0)
    with pytest.raises(RuntimeError, match="in 8 bits, or in 16"):
        ops.gated_dgrad(x, w2, ab[:2], scales, 0)
    with pytest.raises(RuntimeError, match="dab"):
        ops.gated_dx(x, w1, w1)
    with pytest.raises(RuntimeError, match="as many rows"):
        ops.gated_wgrad(torch.zeros(3, 2, 16, device="cuda"), x, F32)
    with pytest.raises(RuntimeError, match="gradients like h"):
        ops.add_rms_norm_bwd(x, x[:2], x, x[0], x[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="int8 codes"):
        ops.mx8_dequantize(ab, scales[:1], F32)


def test_single_rows_without_leading_dims():
    g = _gen(31)
    x = _randn(64, gen=g)
    w1, w3, w2 = _randn(96, 64, gen=g, scale=0.2), _randn(96, 64, gen=g, scale=0.2), _randn(64, 96, gen=g, scale=0.2)
    for checkpoint in ("full", "mx8"):
        leaves = [t.clone().requires_grad_() for t in (x, w1, w3, w2)]
        y = K.gated_ffn(*leaves, checkpoint=checkpoint)
        rows = [t.clone().requires_grad_() for t in (x[None], w1, w3, w2)]
        y2 = K.gated_ffn(*rows, checkpoint=checkpoint)
        assert y.shape == (64,) and torch.equal(y, y2[0])
        for a, b in zip(torch.autograd.grad(y.float().sum(), leaves), torch.autograd.grad(y2.float().sum(), rows)):
            assert torch.equal(a, b.view_as(a))


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are what a call of their own gives."""
    M, D = 67000, 32768
    g = _gen(41)
    tail = _randn(300, D, gen=g)
    x = torch.empty(M, D, device="cuda", dtype=BF).fill_(0.5)
    x[-300:] = tail
    codes, scales = K.mx8_quantize(x)
    want = K.mx8_quantize(tail)
    assert torch.equal(codes[-300:], want[0]) and torch.equal(scales[-300:], want[1])
    y = K.mx8_dequantize(codes, scales)
    assert torch.equal(y[-300:], K.mx8_dequantize(*want))
    del codes, scales, y
    w = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(BF)
    n, h, rstd = ops.add_rms_norm(x, x, w, 1e-5)
    n2, h2, rstd2 = ops.add_rms_norm(tail, tail, w, 1e-5)
    assert torch.equal(n[-300:], n2) and torch.equal(h[-300:], h2)
    dx, _ = ops.add_rms_norm_bwd(n, x, h, w, rstd)
    assert torch.equal(dx[-300:], ops.add_rms_norm_bwd(n2, tail, h2, w, rstd2)[0])
    del dx, n, h, x
    torch.cuda.empty_cache()
    x = torch.empty(70000, 31999, device="cuda", dtype=BF).fill_(0.25)  # rows that begin anywhere
    tail = _randn(8, 31999, gen=g)
    x[-8:] = tail
    codes, scales = K.mx8_quantize(x)
    want = K.mx8_quantize(tail)
    assert torch.equal(codes[-8:], want[0]) and torch.equal(scales[-8:], want[1])
    w = torch.ones(31999, device="cuda", dtype=BF)
    _, _, _, q, scale = ops.add_rms_norm_fp8(x, None, w, 1e-5, False)
    _, _, _, q2, scale2 = ops.add_rms_norm_fp8(tail, None, w, 1e-5, False)
    assert torch.equal(q[-8:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale[-8:], scale2)
    del x, codes, scales, q
    torch.cuda.empty_cache()
    M, H = 70016, 16384  # 2 M H of a and b
    x = torch.zeros(M, 64, device="cuda", dtype=BF)
    x[-256:] = _randn(256, 64, gen=g)
    w1, w3, w2 = _randn(H, 64, gen=g, scale=0.1), _randn(H, 64, gen=g, scale=0.1), _randn(64, H, gen=g, scale=0.01)
    for bits in (16, 8):
        h, ab, scales = ops.gated_mm(x, w1, w3, 0, bits)
        a, b = _products(x[-256:], w1, w3)
        _close(h[-256:], F.silu(a) * b, 1.2 * HALF_STEP[BF])
        # at most 2^-7 or 2^-15 of a block's top, itself below 8 times the root mean square; the sums' own error
        _close(_kept(ab[-256:], scales[-256:]), torch.stack((a, b), 1), 2.0**-4 if bits == 8 else 2.0**-12 + 2.0**-18)
        dab, h = ops.gated_dgrad(x, w2, ab, scales, 0)
        few, h2 = ops.gated_dgrad(x[-256:].contiguous(), w2, ab[-256:].contiguous(), scales[-256:].contiguous(), 0)
        _close(dab[-256:], few.double(), 2 * HALF_STEP[BF])
        assert torch.equal(h[-256:], h2)
        _close(ops.gated_dx(dab, w1, w3)[-256:], ops.gated_dx(dab[-256:].contiguous(), w1, w3).double(), 2 * HALF_STEP[BF])
        del h, ab, dab
    torch.cuda.empty_cache()


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_llama_with_the_fused_block(checkpoint):
    """The model's step on the GPU, fused against separate operators, from the same weights."""
    from autoparallel_b200.models.llama3 import Transformer, llama3_debug

    tokens, labels = (torch.randint(0, 1024, (2, 128), device="cuda", generator=_gen(s)) for s in (1, 2))

    def step(**kw):
        m = Transformer(llama3_debug(**kw))
        m.init_weights(0)
        m = m.to("cuda", BF)
        m.rope_cos, m.rope_sin = m.rope_cos.float(), m.rope_sin.float()
        loss = m(tokens, labels)
        loss.backward()
        return float(loss.detach()), {n: p.grad for n, p in m.named_parameters()}

    loss, grads = step()
    fused, g2 = step(fused_ffn=True, fused_norm=True, ffn_checkpoint=checkpoint)
    # bf16 activations of two layers, rounded at about ten places a layer: each 2^-9 of a value on average
    assert abs(fused - loss) < 20 * 2.0**-9 * abs(loss)
    for n, g in grads.items():
        assert torch.isfinite(g2[n]).all() and float((g2[n].double() - g.double()).norm() / g.double().norm()) < 20 * 2.0**-9 * (1 if checkpoint == "full" else 2), n
