"""Routing to experts on the CPU: the operator's formula against a plain one in 64 bits, its gradient against differences, ties, masks,
refusals, the sharding rules and the MoE model's options."""
import pytest
import torch

import autoparallel_b200.ops as K


def plain(x, top_k, score="softmax", bias=None, num_groups=1, top_groups=1, renormalize=True, scale=1.0):
    """Weights [T, k] and experts of every token, one token at a time, in 64 bits."""
    weights, experts = [], []
    for row in x.double():
        s = (torch.softmax(row, 0) if row.max() > -torch.inf else torch.zeros_like(row)) if score == "softmax" else torch.sigmoid(row)
        c = (row if score == "softmax" else s) + (0 if bias is None else bias.double())
        size = len(row) // num_groups
        take = 2 if score == "sigmoid" else 1
        value = [sum(sorted(c[g * size:(g + 1) * size].tolist(), reverse=True)[:take]) for g in range(num_groups)]
        groups = sorted(range(num_groups), key=lambda g: (-value[g], g))[:top_groups]
        may = [e for g in groups for e in range(g * size, (g + 1) * size)]
        idx = sorted(may, key=lambda e: (-c[e].item(), e))[:top_k]
        w = s[idx]
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        weights.append(w * scale)
        experts.append(idx)
    return torch.stack(weights), torch.tensor(experts)


CASES = [
    dict(top_k=2), dict(top_k=1), dict(top_k=8, renormalize=False, scale=2.5), dict(top_k=5, score="sigmoid"),
    dict(top_k=5, score="sigmoid", renormalize=False), dict(top_k=4, num_groups=4, top_groups=2),
    dict(top_k=6, score="sigmoid", num_groups=4, top_groups=2),
    dict(top_k=3, score="sigmoid", num_groups=16, top_groups=5, scale=0.5), dict(top_k=16),
]


@pytest.mark.parametrize("how", CASES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_formula(how, with_bias):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 16, generator=g)
    bias = torch.randn(16, generator=g) * 0.1 if with_bias else None
    w, idx = K.moe_route(x, bias=bias, **how)
    ref_w, ref_idx = plain(x, bias=bias, **how)
    assert w.dtype == torch.float32 and idx.dtype == torch.long
    assert torch.equal(idx, ref_idx)
    assert torch.allclose(w.double(), ref_w, rtol=1e-5, atol=1e-7)  # 16 fp32 terms: 16 * 2^-24 of the sum


@pytest.mark.parametrize("how", CASES)
def test_gradient_is_the_formulas(how):
    """Against differences in 64 bits of the weights with the experts held."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, 16, generator=g)
    dw = torch.randn(12, how["top_k"], generator=g)
    xg = x.clone().requires_grad_()
    w, idx = K.moe_route(xg, **how)
    (dx,) = torch.autograd.grad(w, xg, dw)

    def value(z):  # sum of dw * weights of the same experts
        s = torch.softmax(z, -1) if how.get("score", "softmax") == "softmax" else torch.sigmoid(z)
        p = s.gather(1, idx)
        p = p / p.sum(-1, keepdim=True) if how.get("renormalize", True) else p
        return (p * how.get("scale", 1.0) * dw.double()).sum(-1)

    z, h = x.double(), 1e-5
    unit = torch.eye(16).double()
    ref = torch.stack([(value(z + h * unit[e]) - value(z - h * unit[e])) / (2 * h) for e in range(16)], -1)
    assert torch.allclose(dx.double(), ref, rtol=1e-4, atol=1e-6)


def test_ties_go_to_the_lower_index():
    x = torch.zeros(3, 8)
    x[1, 5] = x[1, 2] = 1.0
    _, idx = K.moe_route(x, 3)
    assert idx.tolist() == [[0, 1, 2], [2, 5, 0], [0, 1, 2]]
    x[2, 0] = -0.0  # (equal to 0)
    _, idx = K.moe_route(x, 3, num_groups=4, top_groups=2)
    assert idx[2].tolist() == [0, 1, 2]


def test_masked_experts():
    low = torch.finfo(torch.bfloat16).min
    x = torch.tensor([[-torch.inf] * 6, [-torch.inf, 1.0, -torch.inf, 2.0, -torch.inf, -torch.inf], [low] * 5 + [0.0],
                      [low] * 6]).bfloat16()
    for renormalize in (True, False):
        xg = x.float().requires_grad_()
        w, idx = K.moe_route(xg, 3, renormalize=renormalize)
        assert w[0].tolist() == [0, 0, 0] and idx[0].tolist() == [0, 1, 2]
        assert idx[1].tolist() == [3, 1, 0] and w[1, 2] == 0 and abs(w[1].sum().item() - 1) < 1e-6
        assert idx[2].tolist() == [5, 0, 1] and w[2].tolist() == [1, 0, 0]
        assert torch.allclose(w[3], torch.full((3,), 1 / 3 if renormalize else 1 / 6))
        w.sum().backward()
        assert torch.isfinite(xg.grad).all() and (xg.grad[0] == 0).all()
    w, idx = K.moe_route(x.float(), 2, score="sigmoid")
    assert w[0].tolist() == [0, 0] and idx[0].tolist() == [0, 1]
    # a masked expert of a group that stays comes before any expert of a group that does not
    x = torch.full((1, 8), -torch.inf)
    x[0, 6], x[0, 1] = 3.0, 1.0
    _, idx = K.moe_route(x, 2, num_groups=4, top_groups=1)
    assert idx.tolist() == [[6, 7]]


def test_nan_shows():
    x = torch.zeros(2, 4)
    x[1, 2] = torch.nan
    w, idx = K.moe_route(x, 2)
    assert idx[1].tolist() == [2, 0] and w[1].isnan().all() and w[0].tolist() == [0.5, 0.5]


def test_empty_batch_and_leading_dims():
    w, idx = K.moe_route(torch.zeros(0, 8), 2)
    assert w.shape == idx.shape == (0, 2)
    x = torch.randn(2, 3, 8)
    w, idx = K.moe_route(x, 2)
    w2, idx2 = K.moe_route(x.view(6, 8), 2)
    assert torch.equal(w.view(6, 2), w2) and torch.equal(idx.view(6, 2), idx2)


@pytest.mark.parametrize("bad", [
    dict(top_k=0), dict(top_k=9), dict(top_k=2, score="relu"), dict(top_k=2, num_groups=3), dict(top_k=2, num_groups=4, top_groups=5),
    dict(top_k=3, num_groups=4, top_groups=1), dict(top_k=2, num_groups=0), dict(top_k=2, bias=torch.zeros(7)),
    dict(top_k=2, bias=torch.zeros(8, dtype=torch.bfloat16))])
def test_refusals(bad):
    with pytest.raises(ValueError, match="moe_route"):
        K.moe_route(torch.zeros(4, 8), **bad)
    with pytest.raises(ValueError, match="moe_route"):
        K.moe_route(torch.zeros(4, 8, dtype=torch.float16), 2)
    with pytest.raises(ValueError, match="moe_route"):
        K.moe_route(torch.zeros(4, 1025), 2)
    with pytest.raises(ValueError, match="moe_route"):
        K.moe_route(torch.zeros(4, 64), 33)


def test_meta_shapes():
    w, idx = torch.ops.apb200.moe_route(torch.empty(5, 7, 16, device="meta"), None, 3, False, 1, 1, True, 1.0)
    assert w.shape == idx.shape == (5, 7, 3) and w.dtype == torch.float32 and idx.dtype == torch.long
    assert torch.ops.apb200.moe_route_bwd(w, torch.empty(5, 7, 16, device="meta", dtype=torch.bfloat16), idx, False, True,
                                          1.0).dtype == torch.bfloat16


def test_softmax_option_of_the_model_matches_its_own_formula():
    from autoparallel_b200.models.moe import MoEFFN, moe_debug

    torch.manual_seed(0)
    a, b = MoEFFN(moe_debug()), MoEFFN(moe_debug(router_score="softmax"))
    b.load_state_dict(a.state_dict())
    a.router.weight.data.normal_()
    b.router.weight.data.copy_(a.router.weight)
    x = torch.randn(2, 8, 128)
    (wa, ia), (wb, ib) = a.route(x), b.route(x)
    assert torch.equal(ia, ib) and torch.allclose(wa, wb, rtol=1e-5, atol=1e-7)
    c = MoEFFN(moe_debug(router_score="sigmoid", router_groups=4, router_top_groups=2, router_scale=2.5))
    c.router.weight.data.copy_(a.router.weight)
    w, idx = c.route(x)
    assert torch.allclose(w.sum(-1), torch.full((2, 8), 2.5)) and all(len({e // 2 for e in t}) <= 2 for t in idx.view(-1, 2).tolist())
