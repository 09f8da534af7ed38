"""The feed-forward block's operators (ops/ffn_ops.py): formulas, gradients and refusals, on the CPU."""
import math

import pytest
import torch
import torch.nn.functional as F

import autoparallel_b200.ops as K
from autoparallel_b200.ops import ffn_ops as FFN
from autoparallel_b200.ops.library import ops

ACTS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}
EPS = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step of a rounding, relative


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _randn(*shape, dtype=torch.float32, gen=None):
    return torch.randn(*shape, generator=gen).to(dtype)


def _near(got, want, dtype, roundings):
    """``roundings`` of the type (and the fp32 arithmetic behind them, sums of a few dozen terms) relative to the result's size."""
    tol = roundings * EPS[dtype] + 64 * 2.0**-24
    assert got.dtype == dtype and (got.double() - want).abs().max() <= tol * want.abs().max().clamp_min(1e-30), (got.double() - want).abs().max()


# ------------------------------------------------------------------------------------ 8-bit checkpoints
def _mx8_exact(x):
    """The definition, block by block in 64 bits: (codes, scale bytes, values)."""
    *lead, k = x.shape
    rows = x.double().reshape(math.prod(lead), k)
    nb = -(-k // 32)
    codes, byte, values = torch.zeros(rows.shape), torch.zeros(rows.shape[0], nb), torch.zeros(rows.shape, dtype=torch.float64)
    for r in range(rows.shape[0]):
        for j in range(nb):
            v = rows[r, 32 * j:32 * j + 32]
            if not torch.isfinite(v).all():
                byte[r, j], values[r, 32 * j:32 * j + 32] = 255, float("nan")
                continue
            top = float(v.abs().max())
            e = -120
            while e < 127 and 2.0**(e + 1) <= top:
                e += 1
            c = torch.clamp(torch.round(v / 2.0**(e - 6)), -127, 127)
            codes[r, 32 * j:32 * j + 32], byte[r, j], values[r, 32 * j:32 * j + 32] = c, e + 127, c * 2.0**(e - 6)
    return codes.reshape(x.shape), byte.reshape(*lead, nb), values.reshape(x.shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 32), (2, 5, 33), (7, 100), (64,), (0, 40), (3, 0)])
def test_mx8(shape, dtype):
    x = _randn(*shape, dtype=dtype, gen=_gen(3)) * 3
    if x.numel() > 3:
        x.view(-1)[1] = 0.0
        x.view(-1)[2] = 63.9 * x.view(-1)[0]
    codes, scales = K.mx8_quantize(x)
    c, s, v = _mx8_exact(x)
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scales.shape == (*shape[:-1], -(-shape[-1] // 32))
    assert torch.equal(codes.float(), c.float()) and torch.equal(scales.float(), s.float())
    for t in (torch.bfloat16, torch.float32):
        assert torch.equal(K.mx8_dequantize(codes, scales, t).double(), v)
    meta = ops.mx8_quantize(x.to("meta"))
    assert [tuple(m.shape) for m in meta] == [tuple(codes.shape), tuple(scales.shape)] and [m.dtype for m in meta] == [torch.int8, torch.uint8]


def test_16_bit_codes():
    """What "full" keeps of both projections of bf16 operands: the same format with 14 for 6, -112 for -120 and 32767 for 127."""
    x = _randn(5, 70, gen=_gen(8)) * 3
    x[1, :32], x[2, 0], x[3, 40], x[4, 33] = 0, 2.0**-126, float("inf"), float("nan")
    x[1, 32:64] = 0.5  # (nothing in the block above the two that round to 32768)
    x[1, 40], x[1, 41] = 32767.6 * 2.0**-14, -32767.6 * 2.0**-14
    codes, scales = FFN._quantize(x, 16)
    assert codes.dtype == torch.int16 and scales.shape == (5, 3) and scales[1, 0] == 15 and scales[3, 1] == scales[4, 1] == 255
    v = FFN._dequantize(codes, scales, torch.float32)
    assert v[3, 32:64].isnan().all() and v[4, 32:64].isnan().all() and codes[1, 40] == 32767 and codes[1, 41] == -32767
    top = F.pad(x, (0, 26)).unflatten(-1, (3, 32)).abs().amax(-1, keepdim=True).expand(5, 3, 32).flatten(1)[:, :70]
    ok = torch.isfinite(top)
    step = torch.exp2(torch.floor(torch.log2(top[ok].double().clamp_min(2.0**-112))) - 14)
    err = (v[ok].double() - x[ok].double()).abs()
    assert (err <= torch.where(x[ok].abs() > 32767.4 * step, 1.0, 0.5) * step).all()


def test_mx8_of_extreme_values():
    big, tiny, inf = torch.finfo(torch.float32).max, 2.0**-126, float("inf")
    x = torch.zeros(8, 32)
    x[1, 0], x[1, 1] = big, -big
    x[2, 0] = tiny
    x[3, 0] = 2.0**-149
    x[4, 3] = inf
    x[5, 4] = float("nan")
    x[6] = 127.6  # (rounds to 128, which is not held)
    x[7] = torch.arange(32) / 32.0 * 2.0**-125
    codes, scales = K.mx8_quantize(x)
    c, s, v = _mx8_exact(x)
    assert torch.equal(scales.float(), s)
    assert torch.equal(codes.float(), c)
    assert torch.equal(K.mx8_dequantize(codes, scales, torch.float32).double().nan_to_num(nan=7.0), v.nan_to_num(nan=7.0))
    assert codes[6].eq(127).all() and scales[0].item() == 7


# ------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (5, 37), (2, 3, 64), (64,), (0, 16)])
def test_add_rms_norm(shape, dtype):
    g = _gen(1)
    x, r, dy, dh = (_randn(*shape, dtype=dtype, gen=g) for _ in range(4))
    w = _randn(shape[-1], dtype=dtype, gen=g)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = K.add_rms_norm(*leaves, 1e-5)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    hd, wd = h.detach().double().requires_grad_(), w.double().requires_grad_()
    yd = hd * torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * wd
    if not x.numel():
        assert y.shape == x.shape
        return
    _near(y, yd.detach(), dtype, 1)
    assert torch.equal(y, ops.rms_norm(h, w, 1e-5)[0])
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    dx, dw = torch.autograd.grad((yd, hd * 1), (hd, wd), (dy.double(), dh.double()))
    _near(got[0], dx, dtype, 1)
    assert torch.equal(got[0], got[1])
    _near(got[2], dw, dtype, 1)


def test_add_rms_norm_where_one_result_is_used():
    x, r = (_randn(4, 24, gen=_gen(s)).requires_grad_() for s in (1, 2))
    w = torch.ones(24, requires_grad=True)
    y, h = K.add_rms_norm(x, r, w)
    (gx,) = torch.autograd.grad(h.sum(), x)
    assert torch.equal(gx, torch.ones_like(x))
    y, h = K.add_rms_norm(x, r, w)
    got = torch.autograd.grad(y.square().sum(), (x, r, w))
    s = (x + r).detach().requires_grad_()
    want = torch.autograd.grad(ops.rms_norm(s, w, 1e-5)[0].square().sum(), (s, w))
    assert torch.allclose(got[0], want[0], atol=1e-5) and torch.allclose(got[1], want[0], atol=1e-5) and torch.allclose(got[2], want[1], rtol=1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [True, False])
def test_add_rms_norm_fp8(residual, dtype):
    g = _gen(5)
    x = _randn(6, 40, dtype=dtype, gen=g)
    r = _randn(6, 40, dtype=dtype, gen=g) if residual else None
    x[3] = 0
    if residual:
        r[3] = 0
    w = _randn(40, dtype=dtype, gen=g)
    y, h, q, scale = K.add_rms_norm_fp8(x, r, w)
    want_y, want_h = K.add_rms_norm(x, r if residual else torch.zeros_like(x), w)
    assert torch.equal(y, want_y) and torch.equal(h, want_h) and (residual or h is x)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (6, 1) and scale[3].item() == 1.0 and not q[3].float().any()
    hd = h.double()
    yd = hd * torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    # half a step of e4m3 (2^-4 relative, 2^-10 in the lowest binade), in units of the scale
    err = (q.double() * scale.double() - yd).abs()
    assert (err <= 1.001 * torch.maximum(yd.abs() * 2.0**-4, scale.double() * 2.0**-10)).all()
    assert ((yd.abs().amax(-1, keepdim=True) / 448 - scale.double()).abs()[:3] <= 2.0**-20 * scale.double()[:3]).all()
    none = K.add_rms_norm_fp8(x, r, w, keep=False)
    assert none[0] is None and torch.equal(none[2].float(), q.float()) and torch.equal(none[3], scale) and torch.equal(none[1], h)
    # the gradient reaches the operands through the 16-bit result
    leaves = [t.clone().requires_grad_() for t in (x, r, w) if t is not None]
    y, h, q, scale = K.add_rms_norm_fp8(leaves[0], leaves[1] if residual else None, leaves[-1])
    assert not q.requires_grad and not scale.requires_grad
    dy = _randn(6, 40, dtype=dtype, gen=g)
    got = torch.autograd.grad(y, leaves, dy)
    h2 = want_h.clone().requires_grad_()
    w2 = w.clone().requires_grad_()
    want = torch.autograd.grad(ops.rms_norm(h2, w2, 1e-5)[0], (h2, w2), dy)
    assert all(torch.equal(a, want[0]) for a in got[:-1]) and torch.equal(got[-1], want[1])


# ------------------------------------------------------------------------------------ gated block
@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("shape,hidden,out", [((5, 24), 40, 24), ((2, 3, 8), 33, 16), ((1, 1), 1, 1), ((12,), 20, 12)])
def test_gated_ffn(shape, hidden, out, act, checkpoint):
    g = _gen(9)
    x = _randn(*shape, gen=g)
    w1, w3, w2 = _randn(hidden, shape[-1], gen=g), _randn(hidden, shape[-1], gen=g), _randn(out, hidden, gen=g)
    dy = _randn(*shape[:-1], out, gen=g)
    leaves = [t.clone().requires_grad_() for t in (x, w1, w3, w2)]
    y = K.gated_ffn(*leaves, act=act, checkpoint=checkpoint)
    d = [t.double() for t in (x, w1, w3, w2)]
    a, b = d[0] @ d[1].t(), d[0] @ d[2].t()
    _near(y.detach(), (ACTS[act](a) * b) @ d[3].t(), torch.float32, 2)
    assert torch.equal(y, K.gated_ffn(x, w1, w3, w2, act=act))
    got = torch.autograd.grad(y, leaves, dy)
    # the gradients at what was kept
    xk = d[0]
    if checkpoint == "mx8":
        xk = _mx8_exact(x)[2]
        _, ab, scales = ops.gated_mm(x, w1, w3, FFN.ACTS[act], 8)
        a, b = K.mx8_dequantize(ab, scales, torch.float32).double().unbind(-2)
    a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
    h = ACTS[act](a) * b
    da, db = torch.autograd.grad(h, (a, b), dy.double() @ d[3])
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    want = (da @ d[1] + db @ d[2], flat(da).t() @ flat(xk), flat(db).t() @ flat(xk), flat(dy.double()).t() @ flat(h.detach()))
    for u, v in zip(got, want):
        _near(u, v, torch.float32, 4)


@pytest.mark.parametrize("act", sorted(ACTS))
def test_gated_ffn_against_differences(act):
    g = _gen(11)
    x, w1, w3, w2 = (_randn(*s, gen=g).requires_grad_() for s in ((4, 8), (12, 8), (12, 8), (6, 12)))
    d = [t.detach().double() for t in (x, w1, w3, w2)]
    dy = _randn(4, 6, gen=g)
    grads = torch.autograd.grad(K.gated_ffn(x, w1, w3, w2, act=act), (x, w1, w3, w2), dy)

    def f(i, t):
        p = list(d)
        p[i] = p[i] + t
        return (((ACTS[act](p[0] @ p[1].t()) * (p[0] @ p[2].t())) @ p[3].t()) * dy.double()).sum()

    for i, grad in enumerate(grads):
        step = torch.randn(grad.shape, generator=g, dtype=torch.float64)
        diff = (f(i, 1e-5 * step) - f(i, -1e-5 * step)) / 2e-5
        # fp32 products of a few dozen terms: 64 roundings of 2^-24 against the sum of magnitudes; differences: 1e-10 of the third derivative
        assert abs(float((grad.double() * step).sum() - diff)) <= 64 * 2.0**-24 * float((grad.double() * step).abs().sum()) * 4 + 1e-6


def test_gated_block_of_nothing():
    for m, d, h, n in ((0, 8, 16, 8), (3, 0, 16, 8), (3, 8, 0, 8), (3, 8, 16, 0)):
        x, w1, w3, w2 = (torch.randn(*s).requires_grad_() for s in ((m, d), (h, d), (h, d), (n, h)))
        for checkpoint in ("full", "mx8"):
            y = K.gated_ffn(x, w1, w3, w2, checkpoint=checkpoint)
            assert y.shape == (m, n) and not y.any()
            for t, g in zip((x, w1, w3, w2), torch.autograd.grad(y.sum(), (x, w1, w3, w2))):
                assert g.shape == t.shape and not g.any()


def test_what_the_backward_pass_keeps():
    """Bytes held between the passes: x in bf16, a and b in 16 bits and a 32nd of a byte, or all in 33/32 of a byte."""
    x, w1, w3, w2 = (torch.randn(*s).bfloat16().requires_grad_() for s in ((64, 128), (256, 128), (256, 128), (128, 256)))
    held = {}
    for checkpoint in ("full", "mx8"):
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
            K.gated_ffn(x, w1, w3, w2, checkpoint=checkpoint)
        held[checkpoint] = sum(t.numel() * t.element_size() for t in seen if all(t is not w for w in (w1, w3, w2)))
    x, ab = 64 * 128, 64 * 2 * 256
    assert held == {"full": 2 * (x + ab) + ab // 32, "mx8": (x + ab) + (x + ab) // 32}


# ------------------------------------------------------------------------------------ refusals
def _refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_refusals():
    x, w = torch.randn(4, 8), torch.ones(8)
    _refused("not alike", K.add_rms_norm, x, x[:2], w)
    _refused("not alike", K.add_rms_norm, x, x[0], w)
    _refused("not alike", K.add_rms_norm, x, x.bfloat16(), w)
    _refused("expected", K.add_rms_norm, x, x, w[:4])
    _refused("expected", K.add_rms_norm, x, x, w.half())
    _refused("bf16 or fp32", K.add_rms_norm, x.half(), x.half(), w)
    _refused("at most 32768", K.add_rms_norm, torch.zeros(1, 32776), torch.zeros(1, 32776), torch.zeros(32776))
    _refused("D at least 1", K.add_rms_norm, torch.zeros(2, 0), torch.zeros(2, 0), torch.zeros(0))
    _refused("different devices", K.add_rms_norm, x, x.to("meta"), w)
    _refused("leaves out", K.add_rms_norm_fp8, x.clone().requires_grad_(), x, w, keep=False)
    with torch.no_grad():
        K.add_rms_norm_fp8(x.clone().requires_grad_(), x, w, keep=False)
    _refused("bf16 or fp32", K.mx8_quantize, x.double())
    _refused("no dims", K.mx8_quantize, torch.tensor(1.0))
    codes, scales = K.mx8_quantize(x)
    _refused("do not belong", K.mx8_dequantize, codes, scales[:2])
    _refused("expected, not", K.mx8_dequantize, codes.view(torch.uint8), scales)
    _refused("not offered", K.mx8_dequantize, codes, scales, torch.float16)
    w1, w2 = torch.randn(16, 8), torch.randn(8, 16)
    _refused("act is one of", K.gated_ffn, x, w1, w1, w2, act="relu")
    _refused("checkpoint is one of", K.gated_ffn, x, w1, w1, w2, checkpoint="fp8")
    _refused("all bf16 or all fp32", K.gated_ffn, x, w1, w1, w2.bfloat16())
    _refused("all bf16 or all fp32", K.gated_ffn, x.half(), w1.half(), w1.half(), w2.half())
    _refused("expected", K.gated_ffn, x, w1, w1[:8], w2)
    _refused("expected", K.gated_ffn, x, w1, w1, w2.t())
    _refused("expected", K.gated_ffn, x[:, :4], w1, w1, w2)
    _refused("expected", K.gated_ffn, torch.tensor(1.0), w1, w1, w2)
    _refused("different devices", K.gated_ffn, x, w1, w1.to("meta"), w2)
    y = ops.gated_ffn(x.clone().requires_grad_(), w1, w1, w2, 0, 0)[0]
    with pytest.raises(RuntimeError, match="kept nothing"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [0, 8, 16])
def test_meta_shapes(bits, dtype):
    x, w1, w3, w2 = (torch.randn(*s).to(dtype) for s in ((2, 3, 24), (40, 24), (40, 24), (16, 40)))
    for name, args in (("gated_mm", (x, w1, w3, 0, bits)), ("gated_ffn", (x, w1, w3, w2, 0, bits)), ("add_rms_norm", (x, x, x[0, 0], 1e-5)),
                       ("add_rms_norm_fp8", (x, x, x[0, 0], 1e-5, bits > 0)), ("add_rms_norm_fp8", (x, None, x[0, 0], 1e-5, bits > 0))):
        real = getattr(ops, name)(*args)
        meta = getattr(ops, name)(*(t.to("meta") if isinstance(t, torch.Tensor) else t for t in args))
        assert [(tuple(a.shape), a.dtype) for a in real] == [(tuple(a.shape), a.dtype) for a in meta], name
    if bits:
        _, ab, scales = ops.gated_mm(x, w1, w3, 0, bits)
        dy = torch.randn(2, 3, 16).to(dtype)
        real = ops.gated_dgrad(dy, w2, ab, scales, 0)
        meta = ops.gated_dgrad(*(t.to("meta") for t in (dy, w2, ab, scales)), 0)
        assert [(tuple(a.shape), a.dtype) for a in real] == [(tuple(a.shape), a.dtype) for a in meta]
        dab = real[0]
        assert ops.gated_dx(dab.to("meta"), w1.to("meta"), w3.to("meta")).shape == ops.gated_dx(dab, w1, w3).shape
        real, meta = ops.gated_wgrad(dab, x, torch.float32), ops.gated_wgrad(dab.to("meta"), x.to("meta"), torch.float32)
        assert [tuple(a.shape) for a in real] == [tuple(a.shape) for a in meta]


# ------------------------------------------------------------------------------------ planner and model
def _rows(mesh, name, *args):
    from autoparallel_b200.parallel.strategies import rules

    op = getattr(torch.ops.apb200, name).default
    ctx = rules.RuleCtx(mesh, op, args, {}, [a for a in args if isinstance(a, torch.Tensor)], None, op(*args), True)
    found = set()
    for s in rules.get_rule(op)(ctx).strategies:
        outs = s.output_specs if isinstance(s.output_specs, (tuple, list)) else [s.output_specs]
        found.add(tuple(o.placements[0] for o in outs) + tuple(i.placements[0] for i in s.input_specs))
    return found


def test_rules(mesh_1d):
    from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

    S, R, P = Shard, Replicate(), Partial()
    x, w1, w2 = torch.randn(8, 16, 64), torch.randn(256, 64), torch.randn(64, 256)
    assert _rows(mesh_1d, "add_rms_norm", x, x, x[0, 0], 1e-5) == {(R,) * 6, (S(0),) * 5 + (R,), (S(1),) * 5 + (R,)}
    assert _rows(mesh_1d, "add_rms_norm_fp8", x, None, x[0, 0], 1e-5, False) == {
        (R,) * 7, *((R, R, S(i), S(i), S(i), S(i), R) for i in (0, 1))}
    assert _rows(mesh_1d, "add_rms_norm_bwd", x, x, x, x[0, 0], x[..., 0]) == {
        (R,) * 7, *((S(i), P, S(i), S(i), S(i), R, S(i)) for i in (0, 1))}
    assert _rows(mesh_1d, "mx8_quantize", x) == {(R,) * 3, (S(0),) * 3, (S(1),) * 3}
    assert _rows(mesh_1d, "mx8_quantize", w2) == {(R,) * 3, (S(0),) * 3, (S(1),) * 3}
    full = {(R,) * 9, *((S(i), S(i), R, R, R, S(i), R, R, R) for i in (0, 1)), (P, S(3), R, R, R, R, S(0), S(0), S(1)),
            (S(2), R, R, R, R, R, R, R, S(0))}
    assert _rows(mesh_1d, "gated_ffn", x, w1, w1, w2, 0, 16) == full
    assert _rows(mesh_1d, "gated_ffn", x, w1, w1, w2, 0, 8) == {
        (R,) * 9, *((S(i),) * 6 + (R,) * 3 for i in (0, 1)), (P, S(3), S(3), R, R, R, S(0), S(0), S(1)), (S(2), R, R, R, R, R, R, R, S(0))}
    half = torch.randn(128, 64)  # 16 columns a rank: half a block
    assert (P, S(3), S(3), R, R, R, S(0), S(0), S(1)) not in _rows(mesh_1d, "gated_ffn", x, half, half, half.t().contiguous(), 0, 8)
    _, ab, scales = ops.gated_mm(x, w1, w1, 0, 8)
    assert _rows(mesh_1d, "gated_dgrad", x, w2, ab, scales, 0) == {
        (R,) * 6, *((S(i), S(i), S(i), R, S(i), S(i)) for i in (0, 1)), (S(3), S(2), R, S(1), S(3), S(3))}
    dab = torch.randn(8, 16, 2, 256)
    assert _rows(mesh_1d, "gated_dx", dab, w1, w1) == {(R,) * 4, *((S(i), S(i), R, R) for i in (0, 1)), (P, S(3), S(0), S(0)), (S(2), R, S(1), S(1))}
    assert _rows(mesh_1d, "gated_wgrad", dab, x, torch.float32) == {
        (R,) * 4, *((P, P, S(i), S(i)) for i in (0, 1)), (S(0), S(0), S(3), R), (S(1), S(1), R, S(2))}


@pytest.mark.parametrize("bits", [8, 16])
def test_splits_of_the_rules_compute_the_same(bits):
    g = _gen(3)
    x, w1, w3, w2 = (_randn(*s, gen=g) for s in ((4, 6, 24), (128, 24), (128, 24), (16, 128)))
    y, ab, scales, _, _ = ops.gated_ffn(x, w1, w3, w2, 0, bits)
    parts = [ops.gated_ffn(x, a, b, c.contiguous(), 0, bits) for a, b, c in zip(w1.chunk(2), w3.chunk(2), w2.chunk(2, 1))]
    assert torch.allclose(sum(p[0] for p in parts), y, atol=1e-4) and torch.equal(torch.cat([p[1] for p in parts], 3), ab)
    if bits == 8:
        assert torch.equal(torch.cat([p[2] for p in parts], 3), scales)
    dy = _randn(4, 6, 16, gen=g)
    dab, h = ops.gated_dgrad(dy, w2, ab, scales, 0)
    halves = [ops.gated_dgrad(dy, c.contiguous(), a.contiguous(), s.contiguous() if bits == 8 else s, 0)
              for c, a, s in zip(w2.chunk(2, 1), ab.chunk(2, 3), scales.chunk(2, 3) if bits == 8 else (scales, scales))]
    assert torch.allclose(torch.cat([p[0] for p in halves], 3), dab, atol=1e-5) and torch.allclose(torch.cat([p[1] for p in halves], 2), h, atol=1e-5)
    dx = ops.gated_dx(dab, w1, w3)
    assert torch.allclose(sum(ops.gated_dx(d.contiguous(), a, b) for d, a, b in zip(dab.chunk(2, 3), w1.chunk(2), w3.chunk(2))), dx, atol=1e-4)
    dw = ops.gated_wgrad(dab, x, torch.float32)
    rows = [ops.gated_wgrad(d.contiguous(), t.contiguous(), torch.float32) for d, t in zip(dab.chunk(2, 1), x.chunk(2, 1))]
    assert all(torch.allclose(rows[0][i] + rows[1][i], dw[i], atol=1e-4) for i in (0, 1))


def _llama(**kw):
    from autoparallel_b200.models.llama3 import Transformer, llama3_debug

    m = Transformer(llama3_debug(**kw))
    m.init_weights(0)
    return m


def test_model_with_the_fused_block():
    """Same weights, same inputs: the fused forms give the loss and the gradients of the separate operators, with 8-bit checkpoints the same
    loss and gradients of the rounded activations."""
    tokens, labels = (torch.randint(0, 1024, (2, 33), generator=_gen(s)) for s in (1, 2))

    def step(**kw):
        m = _llama(**kw)
        loss = m(tokens, labels)
        loss.backward()
        return loss.detach(), {n: p.grad for n, p in m.named_parameters()}

    loss, grads = step()
    for kw, off in ((dict(fused_ffn=True), 1e-4), (dict(fused_norm=True), 1e-4), (dict(fused_ffn=True, fused_norm=True, ffn_checkpoint="mx8"), 2.0**-6)):
        l2, g2 = step(**kw)
        # (8 bits: a rounding of at most 2^-7 of a block's largest value in each of x, a and b)
        assert abs(float(l2 - loss)) < 1e-5 and all(float((g2[n] - g).norm() / g.norm()) < off for n, g in grads.items()), kw
    with pytest.raises(ValueError, match="ffn_checkpoint is one of"):
        _llama(fused_ffn=True, ffn_checkpoint="fp8")
    with pytest.raises(ValueError, match="needs fused_ffn"):
        _llama(ffn_checkpoint="mx8")


@pytest.mark.parametrize("checkpoint", ["full", "mx8"])
def test_planned_model(mesh_2d, checkpoint):
    from torch.distributed.tensor.placement_types import Replicate, Shard

    from autoparallel_b200 import AutoParallel, ForwardInputs
    from autoparallel_b200.models.llama3 import Transformer, llama3_debug

    with torch.device("meta"):
        model = Transformer(llama3_debug(fused_ffn=True, fused_norm=True, ffn_checkpoint=checkpoint))

    def input_fn():
        return ForwardInputs((torch.randint(0, 1024, (8, 64)),), {"labels": torch.randint(0, 1024, (8, 64))})

    with AutoParallel(model, input_fn, mesh_2d) as ap:
        ap.add_input_constraints([(Shard(0), Replicate())] * 2)
        ap.optimize_placement()
        low = ap.lower()
        names = {str(n.target) for n in low.gm.graph.nodes if n.op == "call_function"}
        for op in ("gated_ffn", "gated_dgrad", "gated_dx", "gated_wgrad", "add_rms_norm", "add_rms_norm_bwd", *(("mx8_dequantize",) if checkpoint == "mx8" else ())):
            assert f"apb200.{op}.default" in names, op


def test_costs(mesh_1d):
    from autoparallel_b200.parallel.cost import compute

    apb = torch.ops.apb200
    m, d, h, n = 10, 64, 96, 32
    ffn = compute._flops(apb.gated_ffn.default, (), [[2, 5, d], [h, d], [h, d], [n, h]], [])
    assert ffn == 2.0 * m * (2 * d * h + h * n)
    back = (compute._flops(apb.gated_dgrad.default, (), [[2, 5, n], [n, h], [2, 5, 2, h], [0]], []) + compute._flops(apb.gated_dx.default, (), [[2, 5, 2, h], [h, d], [h, d]], [])
            + compute._flops(apb.gated_wgrad.default, (), [[2, 5, 2, h], [2, 5, d]], []) + 2.0 * m * n * h)
    assert back == 2 * ffn
    assert compute._flops(apb.gated_mm.default, (), [[2, 5, d], [h, d], [h, d]], []) == 4.0 * m * d * h


# ------------------------------------------------------------------------------------ the extension's C entries, without a GPU
def _entries(code):
    import os
    import subprocess
    import sys

    from autoparallel_b200.ops import build

    if not os.path.exists(build.so_path()):
        pytest.skip("the extension is not built")
    head = f"import ctypes, torch\nso = ctypes.CDLL({build.so_path()!r})\nV, LL, F, N = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float, None\n"
    r = subprocess.run([sys.executable, "-c", head + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout.split()


def test_entries_refuse_what_the_kernels_do_not_take():
    """Bases off a 16-byte boundary, widths and strides that are not whole vectors, rows past the widest: code 3, nothing launched."""
    out = _entries("""
p, bad = V(1 << 20), V((1 << 20) + 8)  # (never read)
norm = [p, p, p, p, p, p, p, p, LL(4), 64, F(1e-5), 1, N]
for i in (0, 1, 2, 3, 4, 6):
    print(so.apb_add_rms_norm(*norm[:i], bad, *norm[i + 1:]))
print(so.apb_add_rms_norm(*norm[:9], 32769, *norm[10:]), so.apb_add_rms_norm(*norm[:9], 0, *norm[10:]))
print(so.apb_add_rms_norm(*norm[:3], N, *norm[4:]), so.apb_add_rms_norm(*norm[:4], N, p, N, p, *norm[8:]))  # a residual without h; no result
back = [p, p, p, p, p, p, p, p, LL(4), 64, 1, 148, N]
for i in (0, 1, 2, 3, 5):
    print(so.apb_add_rms_norm_bwd(*back[:i], bad, *back[i + 1:]))
for f in (so.apb_mx8_quantize, so.apb_mx8_dequantize):
    for i in (0, 2 if f is so.apb_mx8_dequantize else 1):
        a = [p, p, p, LL(4), LL(64), 1, N]
        a[i] = bad
        print(f(*a))
    print(f(p, p, p, LL(1 << 31), LL(33), 1, N))
gated = [p, p, p, p, p, p, 16, 4, 64, 64, LL(64), LL(64), LL(64), 0, p, 148, N]
for i in (0, 1, 2, 3, 4):
    print(so.apb_gemm_gated(*gated[:i], bad, *gated[i + 1:]))
for i in (8, 9):
    print(so.apb_gemm_gated(*gated[:i], 60, *gated[i + 1:]))
for i in (10, 11, 12):
    print(so.apb_gemm_gated(*gated[:i], LL(60), *gated[i + 1:]))
print(so.apb_gemm_gated(*gated[:6], 4, *gated[7:]), so.apb_gemm_gated(*gated[:5], N, *gated[6:]))  # bits; codes without scales
grad = [p, p, p, p, 8, p, p, 4, 64, 64, LL(64), LL(64), 0, p, 148, N]
print(so.apb_gemm_gated_grad(*grad[:4], 0, *grad[5:]), so.apb_gemm_gated_grad(*grad[:3], N, *grad[4:]))
for i in (0, 1, 2, 5, 6):
    print(so.apb_gemm_gated_grad(*grad[:i], bad, *grad[i + 1:]))
dual = [p, p, p, p, p, 4, 64, 64, LL(128), LL(64), LL(64), LL(64), p, 148, N]
for i in (0, 1, 2, 3, 4):
    print(so.apb_gemm_dual(*dual[:i], bad, *dual[i + 1:]))
""")
    assert out == ["3"] * len(out) and len(out) == 6 + 2 + 2 + 5 + 6 + 5 + 2 + 3 + 2 + 2 + 5 + 5, out
    out = _entries("""
p = V(1 << 20)
print(so.apb_add_rms_norm(p, p, p, p, p, p, N, N, LL(0), 64, F(1e-5), 1, N), so.apb_mx8_quantize(p, p, p, LL(0), LL(5), 1, N),
      so.apb_gated_act(p, p, LL(0), 4, 0, 1, N))
so.apb_gemm_set_dynamic_tiles(1)
print(so.apb_gemm_gated(p, p, p, p, p, p, 16, 4, 64, 64, LL(64), LL(64), LL(64), 0, p, 148, N))
""")
    assert out == ["0", "0", "0", "-1"]


def test_workspace_of_the_norm_gradient():
    """A row of partial sums per block; a multiple of eight blocks where rows begin anywhere, so that those of a block begin alike."""
    cases = [(1, 8, 1), (5, 4096, 1), (8192, 4096, 1), (1, 7, 1), (999, 1001, 0), (3, 32767, 0), (100000, 33, 1), (0, 64, 1)]
    out = _entries("f = so.apb_add_rms_norm_bwd_workspace\nf.restype = ctypes.c_longlong\n"
                   f"for rows, d, bf in {cases!r}:\n    print(f(LL(rows), d, bf, 148))")
    for (rows, d, _), n in zip(cases, map(int, out)):
        blocks = n // max(d, 1)
        assert n == blocks * d and (rows == 0) == (n == 0) and blocks <= max(148 * 16, 8) + 8
        if d % 8 and rows:
            assert blocks % 8 == 0
        else:
            assert blocks <= max(rows, 0)


@pytest.mark.parametrize("name", ["add_rms_norm", "add_rms_norm_fp8", "mx8_quantize", "mx8_dequantize", "gated_ffn8", "gated_ffn16"])
def test_registration(name):
    """Schema, fake tensors and the traced gradient agree with the operator."""
    g = _gen(2)
    x, w = _randn(3, 40, gen=g).requires_grad_(), _randn(40, gen=g).requires_grad_()
    w1, w3, w2 = (_randn(*s, gen=g).requires_grad_() for s in ((48, 40), (48, 40), (24, 48)))
    codes, scales = K.mx8_quantize(x.detach())
    args = {"add_rms_norm": (x, x.detach(), w, 1e-5), "add_rms_norm_fp8": (x, None, w, 1e-5, True), "mx8_quantize": (x.detach(),),
            "mx8_dequantize": (codes, scales, torch.float32), "gated_ffn8": (x, w1, w3, w2, 1, 8), "gated_ffn16": (x, w1, w3, w2, 0, 16)}[name]
    op = getattr(ops, name.rstrip("0123456789") if name.startswith("gated") else name).default
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


def test_norm_gradient_without_one_of_the_sum(mesh_1d):
    """``add_rms_norm_bwd`` without ``dh``: the plain norm's gradient, its shapes and its ways to be split."""
    from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

    g = _gen(12)
    for dtype in (torch.bfloat16, torch.float32):
        for shape in ((4, 1), (2, 3, 37), (5, 64)):
            h, dy = (_randn(*shape, dtype=dtype, gen=g) for _ in range(2))
            w = _randn(shape[-1], dtype=dtype, gen=g)
            rstd = ops.rms_norm(h, w, 1e-5)[1]
            got, want = ops.add_rms_norm_bwd(dy, None, h, w, rstd), ops.add_rms_norm_bwd(dy, torch.zeros_like(h), h, w, rstd)
            assert all(torch.allclose(a.float(), b.float(), rtol=2 * EPS[dtype], atol=1e-5) for a, b in zip(got, want))
            meta = ops.add_rms_norm_bwd(dy.to("meta"), None, h.to("meta"), w.to("meta"), rstd.to("meta"))
            assert [(a.shape, a.dtype) for a in meta] == [(a.shape, a.dtype) for a in got]
    S, R, P = Shard, Replicate(), Partial()
    x = torch.randn(8, 16, 64)
    assert _rows(mesh_1d, "add_rms_norm_bwd", x, None, x, x[0, 0], x[..., 0]) == {(R,) * 6, *((S(i), P, S(i), S(i), R, S(i)) for i in (0, 1))}


@pytest.mark.parametrize("k", [256, 257])
def test_mx8_values_of_every_scale(k):
    """Codes from elsewhere may come with any scale byte of the format, and with the code -128."""
    codes = (torch.arange(k) % 256 - 128).to(torch.int8).expand(256, k)
    scales = torch.arange(256).to(torch.uint8).unsqueeze(1).expand(256, -(-k // 32))
    want = codes.double() * torch.exp2(scales[:, :1].double() - 133)
    for dtype in (torch.bfloat16, torch.float32):  # (exact in both but for -2^128)
        got = K.mx8_dequantize(codes, scales, dtype)
        assert got[255].isnan().all() and torch.equal(got[:255].double(), want[:255].masked_fill(want[:255] <= -(2.0**128), -math.inf))


def test_fp16_numbers_under_a_power_of_two():
    """What "full" keeps of both projections of bf16 operands: every value to fp16's half step down to 2^-28 of its block's largest."""
    g = _gen(15)
    x = _randn(6, 70, gen=g) * torch.exp2(torch.randint(-34, 1, (6, 70), generator=g).float())
    x[1, :32], x[2, 32:64], x[3, 40], x[4, 3] = 0, x[2, 32:64] * 2.0**-125, float("inf"), float("nan")
    x[5, 0] = -1.7 * 2.0**127
    codes, scales = FFN._quantize(x, 11)
    assert codes.dtype == torch.float16 and scales.shape == (6, 3) and scales[1, 0] == 15 and scales[3, 1] == scales[4, 0] == 255 and scales[5, 0] == 254
    v = FFN._dequantize(codes, scales, torch.float32)
    assert v[3, 32:64].isnan().all() and v[4, :32].isnan().all()
    top = F.pad(x, (0, 26)).unflatten(-1, (3, 32)).abs().amax(-1, keepdim=True).expand(6, 3, 32).flatten(1)[:, :70].double()
    ok = torch.isfinite(top)
    err, e = (v[ok].double() - x[ok].double()).abs(), torch.floor(torch.log2(top[ok].clamp_min(2.0**-112)))
    # (a last 2^-150: values below fp32's normal numbers)
    assert (err <= torch.maximum(2.0**-11 * x[ok].double().abs(), torch.exp2(e - 39)) + 2.0**-150).all()
    assert (err[x[ok].abs() >= top[ok] * 2.0**-28] <= 2.0**-11 * x[ok].double().abs()[x[ok].abs() >= top[ok] * 2.0**-28] + 2.0**-150).all()


@pytest.mark.parametrize("times", [1, 4096, 2.0**24])
def test_full_keeps_small_values_beside_large_ones(times):
    """One column of every block of 32 is much larger than the others: the gradients of the others' weights are as near as they are without it."""
    g = _gen(16)
    x, dy = _randn(64, 48, dtype=torch.bfloat16, gen=g), _randn(64, 40, dtype=torch.bfloat16, gen=g)
    w1, w3, w2 = _randn(70, 48, gen=g) / 7, _randn(70, 48, gen=g) / 7, _randn(40, 70, gen=g) / 8
    large = torch.arange(70) % 32 == 5
    w1[large] *= times
    w3[large] *= times
    leaves = [t.bfloat16().requires_grad_() for t in (x, w1, w3, w2)]
    got = torch.autograd.grad(K.gated_ffn(*leaves), leaves, dy)
    d = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad((F.silu(d[0] @ d[1].t()) * (d[0] @ d[2].t())) @ d[3].t(), d, dy.double())
    for u, v in ((got[1][~large], want[1][~large]), (got[2][~large], want[2][~large]), (got[3][:, ~large], want[3][:, ~large])):
        # two roundings to bf16 (da, db or h, and the result), each at most 2^-8 and evenly spread: sqrt(2 / 3) 2^-8; what is kept adds 2^-11 of each value at most
        assert float((u.double() - v).norm() / v.norm()) <= math.sqrt(2 / 3) * 2.0**-8 + 2.0**-11


def test_16_bit_whole_numbers_as_a_checkpoint():
    """"mx16": a and b of bf16 operands as whole numbers; of fp32 operands as they are."""
    g = _gen(17)
    for dtype, kept in ((torch.bfloat16, torch.int16), (torch.float32, torch.float32)):
        leaves = [_randn(*s, dtype=dtype, gen=g).requires_grad_() for s in ((5, 24), (40, 24), (40, 24), (16, 40))]
        dy = _randn(5, 16, dtype=dtype, gen=g)
        _, ab, scales = ops.gated_mm(*(t.detach() for t in leaves[:3]), 0, 16)
        assert ab.dtype == kept
        got = torch.autograd.grad(K.gated_ffn(*leaves, checkpoint="mx16"), leaves, dy)
        x, w1, w3, w2 = (t.detach() for t in leaves)
        dab, h = ops.gated_dgrad(dy, w2, ab, scales, 0)
        want = (ops.gated_dx(dab, w1, w3), *ops.gated_wgrad(dab, x, dtype), ops.mm_wgrad(dy, h, dtype))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    m = _llama(fused_ffn=True, ffn_checkpoint="mx16")
    assert m.layers["0"].feed_forward.checkpoint == "mx16"


def test_entry_of_two_results_refuses_what_it_does_not_take():
    out = _entries("""
p, bad = V(1 << 20), V((1 << 20) + 8)  # (never read)
two = [p, p, p, p, 64, 64, 5, LL(128), LL(64), 1, p, 148, N]
for i in (0, 1, 2, 3):
    print(so.apb_gemm_two(*two[:i], bad, *two[i + 1:]))
for i in (4, 5):
    print(so.apb_gemm_two(*two[:i], 60, *two[i + 1:]), so.apb_gemm_two(*two[:i], 0, *two[i + 1:]))
print(so.apb_gemm_two(*two[:6], 0, *two[7:]), so.apb_gemm_two(*two[:4], 1 << 30, *two[5:]))
for i in (7, 8):
    print(so.apb_gemm_two(*two[:i], LL(60), *two[i + 1:]))
""")
    assert out == ["3"] * 12, out
    out = _entries("p = V(1 << 20)\nso.apb_gemm_set_dynamic_tiles(1)\nprint(so.apb_gemm_two(p, p, p, p, 64, 64, 5, LL(128), LL(64), 1, p, 148, N))")
    assert out == ["-1"]


def test_gradients_of_both_projections_are_tensors_of_their_own():
    dw1, dw3 = ops.gated_wgrad(torch.randn(5, 2, 16), torch.randn(5, 8), torch.float32)
    assert dw1.untyped_storage().data_ptr() != dw3.untyped_storage().data_ptr() and dw1.untyped_storage().nbytes() == 16 * 8 * 4


def test_norm_gradient_entry_needs_a_status_word():
    """A wait that runs out is recorded there, so the entry launches nothing without one."""
    out = _entries("""
p = V(1 << 20)  # (never read)
for d in (64, 63, 32768):
    print(so.apb_add_rms_norm_bwd(p, p, p, p, p, p, p, p, LL(4), d, 1, 148, N, N, 0), so.apb_add_rms_norm_bwd(p, N, p, p, p, p, p, p, LL(4), d, 1, 148, N, N, 0))
""")
    assert out == ["3"] * 6, out


@pytest.mark.parametrize("act", sorted(ACTS))
def test_activations_against_64_bits(act):
    """Value and derivative of the formulas, relative to their terms, at single values (a sum over a tensor hides 1e-5 of one)."""
    a = torch.linspace(-9, 9, 2001)
    d = a.double().requires_grad_()
    s = {"silu": lambda t: torch.sigmoid(t), "gelu": lambda t: 0.5 * torch.erfc(-t * 0.5**0.5),
         "gelu_tanh": lambda t: torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (t + 0.044715 * t**3))}[act](d)
    (dv,) = torch.autograd.grad((d * s).sum(), d)
    s, d = s.detach(), d.detach()
    # a few roundings, and those of an exponential's argument, which are that much of the value: |u| of gelu_tanh, a^2 / 2 and a constant of gelu
    tol = (32 + 5 * {"silu": d.abs(), "gelu": d.square(), "gelu_tanh": (1.6 * d * (1 + 0.044715 * d * d)).abs()}[act]) * 2.0**-24
    v, slope = FFN._act(FFN.ACTS[act], a)
    assert bool(((v.double() - d * s).abs() <= tol * (d * s).abs()).all())
    assert bool(((slope.double() - dv).abs() <= tol * (s + (dv - s).abs())).all())


@pytest.mark.parametrize("bits", [8, 11, 16])
def test_splits_of_bf16_codes_compute_the_same(bits):
    """The hidden dim in whole blocks: codes and scales of the parts are parts of the whole's, and so is what is made of them."""
    g = _gen(18)
    x, w1, w3, w2 = (_randn(*s, dtype=torch.bfloat16, gen=g) for s in ((4, 6, 24), (128, 24), (128, 24), (16, 128)))
    dy = _randn(4, 6, 16, dtype=torch.bfloat16, gen=g)
    h, ab, scales = ops.gated_mm(x, w1, w3, 1, bits)
    parts = [ops.gated_mm(x, a, b, 1, bits) for a, b in zip(w1.chunk(2), w3.chunk(2))]
    for i, whole in enumerate((h, ab, scales)):
        assert torch.equal(torch.cat([p[i] for p in parts], -1), whole)
    dab, h = ops.gated_dgrad(dy, w2, ab, scales, 1)
    halves = [ops.gated_dgrad(dy, c, p[1], p[2], 1) for c, p in zip(w2.chunk(2, 1), parts)]
    # (dh is a product of its own in the parts: a sum of 16 terms in another order, then a rounding to bf16 that may fall the other way)
    for i, whole in enumerate((dab, h)):
        part = torch.cat([p[i] for p in halves], -1).float()
        assert bool(((part - whole.float()).abs() <= 2.0**-7 * whole.float().abs() + 2.0**-20).all())


def test_rules_of_fp16_numbers(mesh_1d):
    from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

    S, R, P = Shard, Replicate(), Partial()
    for hidden, split in ((256, True), (128, False)):  # 32 and 16 columns a rank
        x, w1, w2 = torch.randn(8, 16, 64).bfloat16(), torch.randn(hidden, 64).bfloat16(), torch.randn(64, hidden).bfloat16()
        rows = _rows(mesh_1d, "gated_ffn", x, w1, w1, w2, 0, 11)
        assert ((P, S(3), S(3), R, R, R, S(0), S(0), S(1)) in rows) == split and (S(0), S(0), S(0), R, R, S(0), R, R, R) in rows
        _, ab, scales = ops.gated_mm(x, w1, w1, 0, 11)
        assert ((S(3), S(2), R, S(1), S(3), S(3)) in _rows(mesh_1d, "gated_dgrad", x, w2, ab, scales, 0)) == split
