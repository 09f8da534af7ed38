"""MXFP4 on the CPU: the format against a plain one in 64 bits, layout, gradients, refusals, sharding rules and the planned MoE model."""
import math

import pytest
import torch

import autoparallel_b200.ops as K
from autoparallel_b200.ops import mx4_ops

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def plain_round(x):
    """Every value of the last dim's blocks of 32 to the nearest that the block can hold, value by value, in 64 bits."""
    out = torch.zeros(x.shape, dtype=torch.float64)
    rows, k = x.reshape(-1, x.shape[-1]).double(), x.shape[-1]
    flat = out.view(-1, k)
    for r in range(rows.shape[0]):
        for j in range(0, k, 32):
            block = rows[r, j:j + 32]
            if not torch.isfinite(block).all():
                flat[r, j:j + 32] = math.nan
                continue
            top = block.abs().max().item()
            unit = 2.0 ** max(min((math.frexp(top)[1] - 1 if top > 0 else -200) - 2, 127), -127)
            for i, v in enumerate((block / unit).tolist()):
                d = (GRID - min(abs(v), 6.0)).abs()
                near = (d == d.min()).nonzero().flatten().tolist()
                flat[r, j + i] = math.copysign(GRID[next((c for c in near if c % 2 == 0), near[0])].item() * unit, v)
    return out


@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (130, 100), (2, 3, 64), (2, 129, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rounding(shape, dtype):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[:-1] + (1,), generator=g))).to(dtype)
    want = plain_round(x)
    assert torch.equal(K.mx4_round(x).double(), want)
    codes, scales = K.mx4_quantize(x)
    assert codes.shape == (*shape[:-1], mx4_ops.padded(shape[-1]) // 2) and scales.shape == (*shape[:-2], *mx4_ops.scale_shape(*shape[-2:]))
    assert torch.equal(K.mx4_dequantize(codes, scales, shape[-1], torch.float32).double(), want)
    xt = x.transpose(-1, -2).contiguous()
    assert torch.equal(K.mx4_round(xt, -2), K.mx4_round(x).transpose(-1, -2))
    assert all(torch.equal(p, q) for p, q in zip(K.mx4_quantize(xt.transpose(-1, -2)), (codes, scales), strict=True))


def test_ties_range_and_broken_blocks():
    x = torch.zeros(8, 32)
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0])  # unit 1: ties to the even code
    x[1, :3] = torch.tensor([7.9, -7.9, 5.0])                              # beyond 6: 6
    x[2, 0], x[3, 0] = math.inf, math.nan
    x[4, :2] = torch.tensor([2.0**-149, 2.0**-130])                        # scale 2^-127 at least
    x[5, 0] = torch.finfo(torch.float32).max
    x[6, :2] = torch.tensor([4.0, -0.0])
    y = K.mx4_round(x)
    assert y[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 4.0]
    assert y[1, :3].tolist() == [6.0, -6.0, 4.0]
    assert y[2].isnan().all() and y[3].isnan().all()
    assert y[4, 0] == 0 and y[4, 1] == 0
    assert y[5, 0] == 6 * 2.0**125 and (y[7] == 0).all()
    codes, scales = K.mx4_quantize(x)
    e = mx4_ops.untile_scales(scales, 8, 1)[:, 0].tolist()
    assert e == [127, 127, 255, 255, 0, 252, 127, 0]
    assert (codes[2] == 0).all() and (codes[3] == 0).all()
    # past the matrix the scales are 2^0
    assert (mx4_ops.untile_scales(scales, 128, 4)[8:] == 127).all() and (mx4_ops.untile_scales(scales, 128, 4)[:, 1:] == 127).all()


def test_scale_tiles():
    """Row r, block j lies at [r / 128, j / 4, (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4]."""
    r, j = 300, 9
    e = torch.arange(r * j).remainder(251).to(torch.uint8).view(r, j)
    t = mx4_ops.tile_scales(e)
    assert t.shape == (3, 3, 512)
    for row in (0, 31, 32, 127, 128, 299):
        for blk in range(j):
            assert t[row // 128, blk // 4, row % 32 * 16 + row % 128 // 32 * 4 + blk % 4] == e[row, blk]
    assert torch.equal(mx4_ops.untile_scales(t, r, j), e)


@pytest.mark.parametrize("lead,m,n,k", [((), 5, 7, 33), ((), 1, 130, 64), ((3,), 4, 9, 96)])
def test_products(lead, m, n, k):
    torch.manual_seed(0)
    x, w = torch.randn(*lead, m, k), torch.randn(*lead, n, k)
    want = plain_round(x) @ plain_round(w).transpose(-1, -2)
    a, b = K.mx4_quantize(x), K.mx4_quantize(w)
    tol = dict(rtol=k * 2.0**-23, atol=k * 2.0**-23 * want.abs().max().item())  # k fp32 additions
    for y in (K.mx4_mm(*a, *b, out_dtype=torch.float32), K.mx4_linear(x, *b), K.mx4_matmul(x, w),
              K.mx4_matmul(x, w.transpose(-1, -2).contiguous(), trans_b=False)):
        assert y.dtype == torch.float32 and torch.allclose(y.double(), want, **tol)
    if not lead:
        y = K.mx4_linear(x.view(1, m, 1, k), *b, out_dtype=torch.bfloat16)
        assert y.shape == (1, m, 1, n) and y.dtype == torch.bfloat16
        assert K.mx4_linear(x[0], *b).shape == (n,)


@pytest.mark.parametrize("lead,trans_b", [((), True), ((), False), ((2,), True), ((2,), False)])
def test_gradients_go_straight_through(lead, trans_b):
    torch.manual_seed(0)
    m, n, k = 6, 10, 40
    x = torch.randn(*lead, m, k, requires_grad=True)
    w = torch.randn(*lead, *((n, k) if trans_b else (k, n)), requires_grad=True)
    dy = torch.randn(*lead, m, n)
    dx, dw = torch.autograd.grad(K.mx4_matmul(x, w, trans_b=trans_b), (x, w), dy)
    xq, wq = plain_round(x.detach()), plain_round(w.detach() if trans_b else w.detach().transpose(-1, -2))
    want_dw = dy.double().transpose(-1, -2) @ xq
    assert torch.allclose(dx.double(), dy.double() @ wq, rtol=1e-5, atol=1e-5)
    assert torch.allclose(dw.double(), want_dw if trans_b else want_dw.transpose(-1, -2), rtol=1e-5, atol=1e-5)
    # ... which is the derivative of the product in the rounded operands
    xd, wd = xq.clone().requires_grad_(), wq.clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda p, q: p @ q.transpose(-1, -2), (xd, wd))
    ref = torch.autograd.grad(xd @ wd.transpose(-1, -2), xd, dy.double())[0]
    assert torch.allclose(dx.double(), ref, rtol=1e-5, atol=1e-5)
    codes, scales = K.mx4_quantize(w.detach() if trans_b else w.detach().transpose(-1, -2))
    (dl,) = torch.autograd.grad(K.mx4_linear(x, codes, scales), x, dy)
    assert torch.allclose(dl.double(), ref, rtol=1e-5, atol=1e-5)
    assert torch.allclose(K.mx4_mm_values(dy, codes, scales, k).double(), ref, rtol=1e-5, atol=1e-5)
    (dr,) = torch.autograd.grad(K.mx4_round(x), x, torch.ones_like(x))
    assert (dr == 1).all()


def test_refusals():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    codes, scales = K.mx4_quantize(w)
    for call in (
        lambda: K.mx4_quantize(x.half()), lambda: K.mx4_quantize(x[0]), lambda: K.mx4_round(x, 0 - 3), lambda: K.mx4_round(x.long()),
        lambda: K.mx4_dequantize(codes, scales, 100), lambda: K.mx4_dequantize(codes, scales[:, :0]),
        lambda: K.mx4_dequantize(codes.int(), scales),
        lambda: K.mx4_dequantize(codes, scales, dtype=torch.float16), lambda: K.mx4_linear(x[:, :32], codes, scales),
        lambda: K.mx4_linear(x.double(), codes, scales), lambda: K.mx4_linear(x, codes, scales, out_dtype=torch.float16),
        lambda: K.mx4_linear(x, codes, scales[..., :100]), lambda: K.mx4_linear(x, codes[None], scales[None]),
        lambda: K.mx4_matmul(x, w, trans_b=False), lambda: K.mx4_matmul(x, w[None]), lambda: K.mx4_matmul(x.half(), w.half()),
        lambda: K.mx4_mm_values(x, codes, scales), lambda: K.mx4_mm_values(x[:, :8], codes, scales, 100),
        lambda: K.mx4_mm_values(x[:, :8], codes[None], scales[None]),
        lambda: K.mx4_mm(codes, scales, codes[None], scales[None]), lambda: K.mx4_mm(codes, scales, *K.mx4_quantize(w[:, :32])),
    ):
        with pytest.raises(ValueError, match="mx4_"):
            call()


def test_empty_operands():
    codes, scales = K.mx4_quantize(torch.zeros(0, 64))
    assert codes.shape == (0, 32) and scales.shape == (0, 1, 512)
    assert K.mx4_linear(torch.zeros(3, 64), codes, scales).shape == (3, 0)
    assert K.mx4_linear(torch.zeros(0, 64), *K.mx4_quantize(torch.ones(5, 64))).shape == (0, 5)
    assert (K.mx4_matmul(torch.zeros(3, 0), torch.zeros(5, 0)) == 0).all()


def _strategies(ap, op):
    node = next(n for n in ap.joint.gm.graph.nodes if n.op == "call_function" and n.target is op)
    found = set()
    for s in ap.sharding_optimizer.strats[node].strategies:
        outs = s.output_specs if isinstance(s.output_specs, (tuple, list)) else [s.output_specs]
        found.add(tuple(o.placements[0] for o in outs) + tuple(i.placements[0] for i in s.input_specs))
    return found


def test_rules(mesh_1d):
    import torch.nn as nn
    from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

    from autoparallel_b200 import AutoParallel

    S, R, P = Shard, Replicate(), Partial()

    class M(nn.Module):
        def __init__(self, k):
            super().__init__()
            self.w = nn.Parameter(torch.empty(64, k))
            self.e = nn.Parameter(torch.empty(8, 64, 32))
            self.register_buffer("bias", torch.zeros(32))

        def forward(self, x):
            y = K.mx4_matmul(x, self.w)                                        # [16, 8, 64]
            z = K.mx4_matmul(y.reshape(8, 16, 64), self.e, trans_b=False)      # [8, 16, 32]
            w, _ = K.moe_route(z, 4, score="sigmoid", bias=self.bias)
            return w.sum()

    apb = torch.ops.apb200
    for k, whole in ((256, True), (128, False)):  # 8 ranks: 32 columns each, or half a block
        with torch.device("meta"):
            m = M(k)
        with AutoParallel(m, lambda: torch.randn(16, 8, k), mesh_1d) as ap:
            node = next(n for n in ap.joint.gm.graph.nodes if n.op == "call_function" and n.target is apb.mx4_matmul.default)
            assert tuple(node.args[1].meta["val"].shape) == (64, k)
            found = _strategies(ap, apb.mx4_matmul.default)
            assert {(S(0), S(0), R), (S(1), S(1), R), (S(2), R, S(0)), (R, R, R)} <= found
            assert ((P, S(2), S(1)) in found) == whole
            found = _strategies(ap, apb.moe_route.default)
            assert (S(0), S(0), S(0), R) in found and (S(1), S(1), S(1), R) in found and not any(S(2) in f for f in found)
            assert (S(0),) * 4 in _strategies(ap, apb.moe_route_bwd.default)
            assert any(n.target is apb.mx4_round.default for n in ap.joint.gm.graph.nodes if n.op == "call_function")
            ap.add_input_constraints([(Shard(0),)])
            ap.optimize_placement()
            ap.lower()


def test_rules_of_codes(mesh_1d):
    from torch.distributed.tensor.placement_types import Partial, Replicate, Shard

    from autoparallel_b200.parallel.strategies import rules

    S, R, P = Shard, Replicate(), Partial()
    apb = torch.ops.apb200

    def found(op, rule, *args):
        out = op(*args)
        ctx = rules.RuleCtx(mesh_1d, op, args, {}, [a for a in args if isinstance(a, torch.Tensor)], None, out, True)
        rows = set()
        for s in rule(ctx).strategies:
            outs = s.output_specs if isinstance(s.output_specs, (tuple, list)) else [s.output_specs]
            rows.add(tuple(o.placements[0] for o in outs) + tuple(i.placements[0] for i in s.input_specs))
        return rows

    w = torch.randn(1024, 1024)
    codes, scales = apb.mx4_quantize(w)
    a, sa = apb.mx4_quantize(w[:64])
    assert found(apb.mx4_quantize.default, rules._mx4_quantize, w) == {(R,) * 3, (S(0),) * 3, (S(1),) * 3}
    assert found(apb.mx4_quantize.default, rules._mx4_quantize, w[:64]) == {(R,) * 3, (S(1),) * 3}
    assert found(apb.mx4_dequantize.default, rules._mx4_dequantize, codes, scales, 1024, torch.float32) == {(R,) * 3, (S(0),) * 3}
    assert found(apb.mx4_mm.default, rules._mx4_mm, a, sa, codes, scales, torch.float32) == {
        (R,) * 5, (S(1), R, R, S(0), S(0)), (P, S(1), S(1), S(1), S(1))}
    assert found(apb.mx4_linear.default, rules._mx4_linear, w[:64], codes, scales, torch.float32) == {
        (R,) * 4, (S(0), S(0), R, R), (S(1), R, S(0), S(0)), (P, S(1), S(1), S(1))}
    assert found(apb.mx4_mm_values.default, rules._mx4_mm_values, w[:64], codes, scales, 1024, torch.float32) == {
        (R,) * 4, (S(0), S(0), R, R), (P, S(1), S(0), S(0))}
    e = torch.randn(8, 16, 64)
    ce, se = apb.mx4_quantize(e)
    assert found(apb.mx4_linear.default, rules._mx4_linear, e, ce, se, torch.float32) == {(R,) * 4, (S(0),) * 4, (S(1), S(1), R, R)}
    # a split that the rules offer computes the same: rows and columns in whole tiles, the contraction in whole blocks
    parts = [apb.mx4_quantize(p.contiguous()) for p in w.chunk(8, 1)]
    assert torch.equal(torch.cat([p[0] for p in parts], 1), codes) and torch.equal(torch.cat([p[1] for p in parts], 1), scales)


def test_planned_moe_model_with_4_bit_experts(mesh_1d):
    from torch.distributed.tensor.placement_types import Shard

    from autoparallel_b200 import AutoParallel, ForwardInputs
    from autoparallel_b200.models.moe import MoETransformer, moe_debug

    for mode in ("planner", "local_map"):
        cfg = moe_debug(expert_mode=mode, expert_format="mx4", router_score="sigmoid", router_groups=4, router_top_groups=2,
                        router_scale=2.5, ep_axis="dp")
        with torch.device("meta"):
            model = MoETransformer(cfg)

        def input_fn():
            return ForwardInputs((torch.randint(0, 512, (8, 64)),), {"labels": torch.randint(0, 512, (8, 64))})

        with AutoParallel(model, input_fn, mesh_1d) as ap:
            ap.add_input_constraints([(Shard(0),)] * 2)
            ap.optimize_placement()
            low = ap.lower()
            names = {str(n.target) for n in low.gm.graph.nodes if n.op == "call_function"}
            assert any("moe_route.default" in n for n in names)
    with pytest.raises(ValueError, match="expert_format"):
        MoETransformer(moe_debug(expert_format="fp8"))


def test_layer_with_4_bit_experts_follows_the_16_bit_one():
    """Same weights: the outputs differ by what 4 bits round away (a quarter of a value at most, less on average), the gradients exist
    and are finite."""
    from autoparallel_b200.models.moe import MoEFFN, moe_debug

    torch.manual_seed(0)
    kw = dict(expert_mode="planner", dispatch_blocks=1, capacity_factor=None, router_score="softmax")
    a, b = MoEFFN(moe_debug(**kw)), MoEFFN(moe_debug(expert_format="mx4", **kw))
    a.init_weights(0.1)
    b.load_state_dict(a.state_dict())
    x = torch.randn(2, 16, 128)
    ya, yb = a(x), b(x)
    rel = ((ya - yb).norm() / ya.norm()).item()
    assert 0 < rel < 0.5
    yb.square().mean().backward()
    for name, p in b.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, name


def test_example():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "examples/example_moe_mx4.py", "--steps", "2"], capture_output=True, text=True, timeout=600,
                       cwd=root)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "mx4_matmul" in r.stdout and "served" in r.stdout


@pytest.mark.parametrize("x_shape,w_shape", [((0,), (48, 0)), ((2, 5, 0), (48, 0)), ((2, 3, 64), (0, 64)), ((0, 64), (48, 64)),
                                             ((3, 5, 0), (3, 48, 0)), ((3, 5, 64), (3, 0, 64))])
def test_matrices_of_nothing(x_shape, w_shape):
    x, w = torch.zeros(x_shape, requires_grad=True), torch.zeros(w_shape, requires_grad=True)
    for trans_b in (True, False):
        m = w if trans_b else w.transpose(-1, -2).contiguous()
        y = K.mx4_matmul(x, m, trans_b=trans_b)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert y.shape == (*x_shape[:-1], w_shape[-2]) and dx.shape == x_shape and dw.shape == w_shape
    codes, scales = K.mx4_quantize(w.detach())
    y = K.mx4_linear(x, codes, scales)
    assert (y == 0).all() and torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x_shape
    assert K.mx4_mm_values(y.detach(), codes, scales, x_shape[-1]).shape == x_shape


@pytest.mark.parametrize("lead,m,n,k", [((), 5, 7, 33), ((3,), 4, 9, 96), ((2, 3), 4, 16, 40)])
def test_gradient_of_products_with_values(lead, m, n, k):
    torch.manual_seed(0)
    codes, scales = K.mx4_quantize(torch.randn(*(lead if len(lead) == 1 else ()), n, k))
    values = K.mx4_dequantize(codes, scales, k, torch.float32).double()
    a, dc, x = torch.randn(*lead, m, n, requires_grad=True), torch.randn(*lead, m, k), torch.randn(*lead, m, k, requires_grad=True)
    ad = a.detach().double().requires_grad_()
    (want,) = torch.autograd.grad(ad @ values, ad, dc.double())
    assert torch.autograd.gradcheck(lambda t: t @ values, ad)
    (da,) = torch.autograd.grad(K.mx4_mm_values(a, codes, scales, k), a, dc)
    assert torch.allclose(da.double(), want, rtol=1e-5, atol=1e-5)
    (dx,) = torch.autograd.grad(K.mx4_linear(x, codes, scales), x, a, create_graph=True)
    (da,) = torch.autograd.grad(dx, a, dc)
    assert torch.allclose(da.double(), want, rtol=1e-5, atol=1e-5)
