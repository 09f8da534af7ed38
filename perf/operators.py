"""The operators of a mixture-of-experts layer with 4-bit products, as timed cases: routing tokens to experts, and
microscaled 4-bit floating point (MXFP4: 4-bit E2M1 values, one power-of-two scale for 32 of them along the contraction).

Sizes are those of this repository's models (``models/moe.py``: 64 experts, top-8, d 2048, hidden 1408;
``models/llama3.py``: 4096 and 14336), of its tests, and generic ones around them.

Kinds
  route    scores, choice of experts and gate weights from router logits; with ``grad`` the gradient of the logits too
  quant    quantisation to 4 bits, and the values that the codes stand for
  linear   a projection of activations by weights that are held in 4 bits (serving); ``experts`` > 0: one of every expert
  train    a projection of both operands rounded to 4 bits, with the gradients of a training step (straight through the rounding)

Layout of a 4-bit matrix [R, K]: codes [R, ceil(K / 32) * 16] uint8, two values a byte, the lower one in the low half; scales, the biased
exponent of each 32 values, in tiles of 128 rows x 4 blocks: byte [r / 128][j / 4][r % 32][r / 32 % 4][j % 4] belongs to row r, block j.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
_DT = {"bf16": BF16, "fp32": F32}


# ------------------------------------------------------------------------------------------------ the list
def listed():
    return [
        # one token being decoded, at the MoE model's router: nothing but latency
        {"name": "route_one", "kind": "route", "tokens": 1, "experts": 64, "topk": 8, "score": "softmax", "groups": 1, "top_groups": 1,
         "bias": False, "renorm": True, "scale": 1.0, "dtype": "bf16", "grad": False},
        # one rank's batch of the MoE model in training
        {"name": "route_8k", "kind": "route", "tokens": 8192, "experts": 64, "topk": 8, "score": "softmax", "groups": 1, "top_groups": 1,
         "bias": False, "renorm": True, "scale": 1.0, "dtype": "bf16", "grad": True},
        # many small experts in groups, sigmoid scores, a bias that balances the load, a ragged number of tokens
        {"name": "route_groups", "kind": "route", "tokens": 16383, "experts": 256, "topk": 8, "score": "sigmoid", "groups": 8,
         "top_groups": 4, "bias": True, "renorm": True, "scale": 2.5, "dtype": "fp32", "grad": True},
        # the largest batch: a whole global batch on one GPU, weights of all scores (no renormalisation)
        {"name": "route_large", "kind": "route", "tokens": 131072, "experts": 128, "topk": 6, "score": "softmax", "groups": 1, "top_groups": 1,
         "bias": True, "renorm": False, "scale": 1.0, "dtype": "bf16", "grad": True},
        # fp32 activations with a ragged row count and a last block that is not full
        {"name": "quant_ragged", "kind": "quant", "experts": 0, "rows": 999, "k": 1000, "dtype": "fp32", "transposed": False},
        # all experts' weights as the MoE model holds them ([E, d, h]), blocks along d
        {"name": "quant_experts", "kind": "quant", "experts": 64, "rows": 1408, "k": 2048, "dtype": "bf16", "transposed": True},
        # one token through the up projection of the 8B model's feed-forward block (decoding)
        {"name": "linear_one", "kind": "linear", "experts": 0, "rows": 1, "n": 14336, "k": 4096, "dtype": "bf16"},
        # a few tokens, odd, through its down projection
        {"name": "linear_few", "kind": "linear", "experts": 0, "rows": 17, "n": 4096, "k": 14336, "dtype": "bf16"},
        # a whole sequence of the 8B model through its up projection: the largest product
        {"name": "linear_8k", "kind": "linear", "experts": 0, "rows": 8192, "n": 14336, "k": 4096, "dtype": "bf16"},
        # 64 experts of the MoE model, each with its capacity of 8192 tokens x 8 choices
        {"name": "linear_experts", "kind": "linear", "experts": 64, "rows": 1280, "n": 1408, "k": 2048, "dtype": "bf16"},
        # the shared expert of the MoE model in training, on a short batch with a ragged token count
        {"name": "train_ragged", "kind": "train", "experts": 0, "rows": 999, "n": 1408, "k": 2048, "dtype": "bf16"},
        # the routed experts in training, on 1024 tokens x 8 choices
        {"name": "train_experts", "kind": "train", "experts": 64, "rows": 160, "n": 1408, "k": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("route", "route", "quant", "linear", "linear", "train"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if kind == "route":
        experts = rng.choice((8, 16, 40, 60, 64, 96, 128, 160, 256))
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 4])
        top_groups = rng.randint(max(1, groups // 2), groups)
        topk = rng.randint(1, min(10, top_groups * (experts // groups)))
        tokens = _log(rng, 1, min(131072, 16777216 // experts))
        return {"kind": kind, "tokens": tokens, "experts": experts, "topk": topk, "score": rng.choice(("softmax", "sigmoid")),
                "groups": groups, "top_groups": top_groups, "bias": rng.random() < 0.5, "renorm": rng.random() < 0.7,
                "scale": rng.choice((1.0, 2.5)), "dtype": dtype, "grad": rng.random() < 0.7}
    experts = rng.choice((0, 0, 4, 8, 16, 64))
    if kind == "quant":
        k = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(2, min(16384, 180_000_000 // (k * max(1, experts)))))
        return {"kind": kind, "experts": experts, "rows": rows, "k": k, "dtype": dtype, "transposed": rng.random() < 0.4}
    k, n = _log(rng, 64, 14336), _log(rng, 64, 14336)
    if experts:
        k, n = min(k, 4096), min(n, 4096)
    most = 4.8e11 if kind == "linear" else 2e10  # (products of a case, at most those of the largest listed one of its kind)
    rows = _log(rng, 1, max(2, min(8192, int(most / (float(k) * n * max(1, experts))))))
    if kind == "train":  # (the 16-bit products of the gradients take rows of whole 16 bytes)
        k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
    return {"kind": kind, "experts": experts, "rows": rows, "n": n, "k": k, "dtype": "bf16" if kind == "train" else dtype}


# ------------------------------------------------------------------------------------------------ inputs
def _activations(shape, gen, dtype):
    """Rows of unequal size, with a few channels that are much larger than the rest."""
    x = torch.randn(shape, device="cuda", generator=gen)
    channel = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=gen))
    channel[torch.rand(shape[-1], device="cuda", generator=gen) < 0.01] *= 20.0
    return (x * channel).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dt = _DT[case["dtype"]]
    if case["kind"] == "route":
        T, E, k = case["tokens"], case["experts"], case["topk"]
        s["logits"] = (1.5 * torch.randn(T, E, device="cuda", generator=gen)).to(dt)
        # (a balance bias moves by a fixed step at a time)
        s["b"] = 0.001 * torch.randint(-50, 51, (E,), device="cuda", generator=gen).float() if case["bias"] else None
        s["dw"] = torch.randn(T, k, device="cuda", generator=gen) if case["grad"] else None
        return s
    lead = (case["experts"],) if case["experts"] else ()
    rows, k = case["rows"], case["k"]
    if case["kind"] == "quant":
        if case["transposed"]:
            s["x"] = (0.02 * torch.randn(*lead, k, rows, device="cuda", generator=gen)).to(dt).transpose(-1, -2)
        else:
            s["x"] = _activations((*lead, rows, k), gen, dt)
        return s
    n = case["n"]
    s["x"] = _activations((*lead, rows, k), gen, dt)
    if case["kind"] == "linear":
        w = (torch.randn(*lead, n, k, device="cuda", generator=gen) * k ** -0.5).to(BF16)
        s["codes"], s["scales"] = _pack(*_quantize(w))
    else:  # experts' weights are held [E, K, N], a projection's [N, K]
        w = torch.randn(*((*lead, k, n) if lead else (n, k)), device="cuda", generator=gen) * k ** -0.5
        s["w"] = w.to(dt)
        s["dy"] = torch.randn(*lead, rows, n, device="cuda", generator=gen).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(n):
    """2^n as fp32, -127 <= n <= 127, exactly."""
    n = n.int()
    return torch.where(n > -127, (n + 127) << 23, 1 << 22).int().view(F32)


def _quantize(x):
    """(codes [..., Kp] of one byte each, biased exponents [..., Kp / 32]) of the last dim."""
    k = x.shape[-1]
    xf = torch.nn.functional.pad(x.float(), (0, -k % 32)).unflatten(-1, (-1, 32))
    amax = xf.abs().amax(-1)
    exponent = torch.where(amax > 0, torch.frexp(amax)[1] - 1 - 2, -127).clamp(-127, 127)
    v = xf.abs() * _pow2(-exponent.unsqueeze(-1))
    # how many of the midpoints between neighbouring values lie below; a tie goes to the even code
    code = ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0))
    code = code + 8 * (xf < 0)
    return code.flatten(-2).to(torch.uint8), (exponent + 127).to(torch.uint8)


def _pack(code, exponent):
    """Codes two to a byte, exponents in their tiles (the rest of the last tiles is 2^0)."""
    codes = code[..., 0::2] + 16 * code[..., 1::2]
    r, j = exponent.shape[-2:]
    e = torch.nn.functional.pad(exponent, (0, -j % 4, 0, -r % 128), value=127)
    e = e.unflatten(-2, (-1, 4, 32)).unflatten(-1, (-1, 4))  # [..., R/128, 4, 32, K/128, 4]
    return codes.contiguous(), e.movedim(-2, -4).transpose(-2, -3).reshape(*e.shape[:-5], e.shape[-5], e.shape[-2], 512).contiguous()


def _unpack(codes, scales):
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    e = scales.unflatten(-1, (32, 4, 4)).transpose(-2, -3).movedim(-4, -2).flatten(-2).flatten(-4, -2)
    return code, e[..., : codes.shape[-2], : codes.shape[-1] // 16]


def _values(code, exponent, k):
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=code.device)
    v = table[code.long()].unflatten(-1, (-1, 32))
    return (v * _pow2(exponent.int().unsqueeze(-1) - 127)).flatten(-2)[..., :k]


def _rounded(x):
    return _values(*_quantize(x), x.shape[-1])


def _route_plain(s):
    x = s["logits"].float()
    T, E = x.shape
    k, groups, scale = s["topk"], s["groups"], s["scale"]
    soft = s["score"] == "softmax"
    if soft:
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = x if soft else score
    if s["b"] is not None:
        choice = choice + s["b"]
    if groups > 1:
        of_group = choice.view(T, groups, E // groups).sort(dim=-1, descending=True).values[..., : 1 if soft else 2].sum(-1)
        best = of_group.sort(dim=-1, descending=True, stable=True).indices[:, : s["top_groups"]]
        kept = torch.zeros_like(of_group, dtype=torch.bool).scatter(1, best, True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // groups, 1), -math.inf)
    idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    picked = score.gather(1, idx)
    total = picked.sum(-1, keepdim=True) if s["renorm"] else 1.0
    p = picked / total
    if s["dw"] is None:
        return {"weights": p * scale, "idx": idx}
    g = s["dw"] * scale
    if s["renorm"]:
        g = (g - (g * p).sum(-1, keepdim=True)) / total
    ds = torch.zeros_like(score).scatter(1, idx, g)
    dx = score * (ds - (ds * score).sum(-1, keepdim=True)) if soft else ds * score * (1 - score)
    return {"weights": p * scale, "idx": idx, "dlogits": dx.to(s["logits"].dtype)}


def _plain(s):
    if s["kind"] == "route":
        return _route_plain(s)
    x, dt = s["x"], s["x"].dtype
    if s["kind"] == "quant":
        return _rounded(x).to(dt)
    if s["kind"] == "linear":
        w = _values(*_unpack(s["codes"], s["scales"]), s["k"])
        return (_rounded(x) @ w.transpose(-1, -2)).to(dt)
    w = s["w"].transpose(-1, -2) if s["experts"] else s["w"]  # [.., N, K]
    xq, wq, dy = _rounded(x), _rounded(w), s["dy"].float()
    dw = dy.transpose(-1, -2) @ xq
    return {"y": (xq @ wq.transpose(-1, -2)).to(dt), "dx": (dy @ wq).to(dt), "dw": (dw.transpose(-1, -2) if s["experts"] else dw).to(dt)}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    import autoparallel_b200.ops as K

    if s["kind"] == "route":
        logits = s["logits"].detach().requires_grad_(s["grad"])
        weights, idx = K.moe_route(logits, s["topk"], score=s["score"], bias=s["b"], num_groups=s["groups"], top_groups=s["top_groups"],
                                   renormalize=s["renorm"], scale=s["scale"])
        if not s["grad"]:
            return {"weights": weights, "idx": idx}
        (dx,) = torch.autograd.grad(weights, logits, s["dw"])
        return {"weights": weights.detach(), "idx": idx, "dlogits": dx}
    x = s["x"]
    if s["kind"] == "quant":
        codes, scales = K.mx4_quantize(x)
        return K.mx4_dequantize(codes, scales, s["k"], x.dtype)
    if s["kind"] == "linear":
        return K.mx4_linear(x, s["codes"], s["scales"])
    x, w = x.detach().requires_grad_(), s["w"].detach().requires_grad_()
    y = K.mx4_matmul(x, w, trans_b=not s["experts"])
    dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "route":
        T, E, k = case["tokens"], case["experts"], case["topk"]
        n = T * E * b + T * k * 12 + (E * 4 if case["bias"] else 0)
        return {"bytes": n + (T * E * b + T * k * 4 if case["grad"] else 0), "flops": T * E * 4 * (2 if case["grad"] else 1)}
    m, k, e = case["rows"], case["k"], max(1, case["experts"])
    if case["kind"] == "quant":
        return {"bytes": 2 * e * m * k * b, "flops": 4 * e * m * k}
    n, kp = case["n"], (k + 31) // 32
    if case["kind"] == "linear":
        return {"bytes": e * (m * k * b + m * n * b + n * kp * 17), "flops": 2 * e * m * n * k}
    return {"bytes": 2 * e * b * (m * k + m * n + n * k), "flops": 6 * e * m * n * k}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_round(x):
    """Every value to the nearest of the 16 that its block can hold."""
    k = x.shape[-1]
    lead = x.shape[:-1]
    out = torch.empty(*lead, k, dtype=F64, device=x.device)
    grid = torch.tensor(sorted(_VALUES), dtype=F64, device=x.device)
    for j in range(0, k, 32):
        block = x[..., j : j + 32].double()
        top = block.abs().amax(-1, keepdim=True)
        unit = torch.exp2((torch.frexp(top.clamp_min(2.0**-140)).exponent - 3).clamp(-127, 127).double())
        v = (block.abs() / unit).clamp_max(6.0)
        hi = torch.searchsorted(grid, v.contiguous()).clamp(1, 7)
        below, above = v - grid[hi - 1], grid[hi] - v
        up = (above < below) | ((above == below) & (hi % 2 == 0))
        out[..., j : j + 32] = torch.where(up, grid[hi], grid[hi - 1]) * unit * torch.sign(block)
    return out


def _exact_route(s):
    x = s["logits"].double()
    T, E = x.shape
    soft = s["score"] == "softmax"
    score = torch.softmax(x, -1) if soft else torch.sigmoid(x)
    choice = (x if soft else score) + (0.0 if s["b"] is None else s["b"].double())
    if s["groups"] > 1:
        per = E // s["groups"]
        of_group = torch.topk(choice.view(T, s["groups"], per), 1 if soft else min(2, per), -1).values.sum(-1)
        floor = torch.topk(of_group, s["top_groups"], -1).values[:, -1:]
        choice = torch.where((of_group < floor).repeat_interleave(per, 1), -math.inf, choice)
    idx = torch.argsort(choice, dim=-1, descending=True, stable=True)[:, : s["topk"]]
    one = torch.nn.functional.one_hot(idx, E).double()  # [T, k, E]
    a = torch.einsum("tke,te->tk", one, score)
    w = s["scale"] * (a / a.sum(-1, keepdim=True) if s["renorm"] else a)
    if s["dw"] is None:
        return {"weights": w, "idx": None}
    g = s["dw"].double()
    # d weights / d picked scores, then d scores / d logits
    da = s["scale"] * g
    if s["renorm"]:
        tot = a.sum(-1, keepdim=True)
        da = da / tot - (da * a).sum(-1, keepdim=True) / tot**2
    dscore = torch.einsum("tke,tk->te", one, da)
    if soft:
        dx = score * dscore - score * torch.einsum("te,te->t", score, dscore).unsqueeze(1)
    else:
        dx = dscore * (score - score * score)
    return {"weights": w, "idx": None, "dlogits": dx}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(s)
    x = s["x"]
    if case["kind"] == "quant":
        return _exact_round(x)
    if case["kind"] == "linear":
        byte = s["codes"].long()
        nibble = torch.stack((byte % 16, byte // 16), -1).flatten(-2)
        value = torch.tensor(_VALUES, dtype=F64, device=x.device)[nibble % 8] * (1 - 2 * (nibble // 8))
        r = torch.arange(value.shape[-2], device=x.device).unsqueeze(1)
        j = torch.arange(value.shape[-1] // 32, device=x.device).unsqueeze(0)
        unit = torch.exp2(s["scales"][..., r // 128, j // 4, r % 32 * 16 + r % 128 // 32 * 4 + j % 4].double() - 127)
        w = (value.unflatten(-1, (-1, 32)) * unit.unsqueeze(-1)).flatten(-2)[..., : case["k"]]
        return torch.einsum("...mk,...nk->...mn", _exact_round(x), w)
    w, dy = s["w"].transpose(-1, -2) if case["experts"] else s["w"], s["dy"].double()
    xq, wq = _exact_round(x), _exact_round(w)
    dw = torch.einsum("...mn,...mk->...nk", dy, xq)
    return {"y": torch.einsum("...mk,...nk->...mn", xq, wq), "dx": torch.einsum("...mn,...nk->...mk", dy, wq),
            "dw": dw.transpose(-1, -2) if case["experts"] else dw}
