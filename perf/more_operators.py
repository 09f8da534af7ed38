"""The feed-forward half of a decoder layer, as timed cases: the residual's addition with the norm after it (and its result in 8 bits),
the gated feed-forward block with its gradients, and activations that are held in 8 bits from the forward pass to the backward pass.

Sizes are those of this repository's models (``models/llama3.py``: 4096 and 14336, 8192; ``models/moe.py``: 2048 and 1408), of its
tests, and generic ones around them.

Kinds
  norm    h = x + residual and y = RMSNorm(h); with ``grad`` the gradients of a training step, in which h is used further on too
  norm8   the same with y in e4m3, one scale a row; ``keep``: and y itself, for the weight gradient of a training step
  save    activations to 8 bits and back (int8 codes, one power of two for 32 values along the last dim)
  ffn     (act(x w1^T) * (x w3^T)) w2^T; with ``grad`` the gradients of x and of the weights.  ``checkpoint`` "mx8": between the two
          passes x and both projections are held in 8 bits, which the gradients are made from
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
F8 = torch.float8_e4m3fn
_DT = {"bf16": BF16, "fp32": F32}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the list
def listed():
    return [
        # one token being decoded, at the 8B model's width: nothing but latency
        {"name": "norm_one", "kind": "norm", "rows": 1, "d": 4096, "dtype": "bf16", "grad": False},
        # a sequence of the 8B model in training
        {"name": "norm_8k", "kind": "norm", "rows": 8192, "d": 4096, "dtype": "bf16", "grad": True},
        # fp32 training with a ragged token count and a width that no vector divides
        {"name": "norm_odd", "kind": "norm", "rows": 999, "d": 1001, "dtype": "fp32", "grad": True},
        # a few tokens on their way into an 8-bit product (serving)
        {"name": "norm8_few", "kind": "norm8", "rows": 17, "d": 4096, "dtype": "bf16", "keep": False},
        # a global batch at the 70B model's width, in 8-bit training
        {"name": "norm8_long", "kind": "norm8", "rows": 32768, "d": 8192, "dtype": "bf16", "keep": True},
        # a ragged activation in fp32, whose last blocks are not full
        {"name": "save_ragged", "kind": "save", "rows": 999, "d": 1000, "dtype": "fp32"},
        # one projection of a sequence of the 8B model
        {"name": "save_8k", "kind": "save", "rows": 8192, "d": 14336, "dtype": "bf16"},
        # one token through the 8B model's feed-forward block
        {"name": "ffn_one", "kind": "ffn", "rows": 1, "d": 4096, "hidden": 14336, "act": "silu",
         "checkpoint": "full", "dtype": "bf16", "grad": False},
        # a few tokens, odd, through a narrow one (the MoE model's shared expert)
        {"name": "ffn_few", "kind": "ffn", "rows": 17, "d": 2048, "hidden": 1408, "act": "gelu_tanh",
         "checkpoint": "full", "dtype": "bf16", "grad": False},
        # a short ragged batch of the shared expert in training, activations in 8 bits
        {"name": "ffn_short", "kind": "ffn", "rows": 999, "d": 2048, "hidden": 1408, "act": "silu",
         "checkpoint": "mx8", "dtype": "bf16", "grad": True},
        # a sequence of the 8B model in training
        {"name": "ffn_8k", "kind": "ffn", "rows": 8192, "d": 4096, "hidden": 14336, "act": "silu",
         "checkpoint": "full", "dtype": "bf16", "grad": True},
        # the same with its activations in 8 bits
        {"name": "ffn_8k_mx8", "kind": "ffn", "rows": 8192, "d": 4096, "hidden": 14336, "act": "gelu",
         "checkpoint": "mx8", "dtype": "bf16", "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm8", "save", "ffn", "ffn", "ffn"))
    if kind == "ffn":  # rows of whole 16 bytes, as projections have them
        d, hidden = (max(8, _log(rng, 64, top) // 8 * 8) for top in (4096, 14336))
        grad = rng.random() < 0.6
        rows = _log(rng, 1, max(2, min(16384, int(4.8e11 / (d * hidden)))))
        return {"kind": kind, "rows": rows, "d": d, "hidden": hidden, "act": rng.choice(("silu", "silu", "gelu", "gelu_tanh")),
                "checkpoint": rng.choice(("full", "mx8")) if grad else "full", "dtype": "bf16", "grad": grad}
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    d = _log(rng, 64, 16384)
    if rng.random() < 0.7:
        d = d // 8 * 8
    most = 58_000_000 if kind == "save" else 100_000_000
    case = {"kind": kind, "rows": _log(rng, 1, max(2, min(65536, most // d))), "d": d, "dtype": dtype}
    if kind == "norm":
        return {**case, "grad": rng.random() < 0.6}
    return {**case, "keep": rng.random() < 0.5} if kind == "norm8" else case


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
    dt, rows, d = _DT[case["dtype"]], case["rows"], case["d"]
    s["x"] = _activations((rows, d), gen, dt)
    if case["kind"] in ("norm", "norm8"):
        s["residual"] = _activations((rows, d), gen, dt)
        s["w"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dt)
        if case.get("grad"):
            s["dy"], s["dh"] = (torch.randn(rows, d, device="cuda", generator=gen).to(dt) for _ in range(2))
    elif case["kind"] == "ffn":
        h = case["hidden"]
        for name, shape in (("w1", (h, d)), ("w3", (h, d)), ("w2", (d, h))):
            s[name] = (torch.randn(*shape, device="cuda", generator=gen) * shape[1] ** -0.5).to(dt)
        if case["grad"]:
            s["dy"] = torch.randn(rows, d, device="cuda", generator=gen).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _norm_plain(s):
    dt = s["x"].dtype
    h = (s["x"].float() + s["residual"].float()).to(dt)
    hf, w = h.float(), s["w"].float()
    r = 1 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    n = hf * r
    y = n * w
    if s["kind"] == "norm8":
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top < 2.0**-100, 1.0, top / 448)
        out = {"h": h, "q": (y / scale).clamp(-448, 448).to(F8), "scale": scale}
        return {**out, "y": y.to(dt)} if s["keep"] else out
    if not s["grad"]:
        return {"y": y.to(dt), "h": h}
    dy = s["dy"].float()
    g = dy * w
    dx = (s["dh"].float() + r * (g - n * (g * n).mean(-1, keepdim=True))).to(dt)
    return {"y": y.to(dt), "h": h, "dx": dx, "dresidual": dx, "dw": (dy * n).sum(0).to(dt)}


def _held(x):
    """The values that 8 bits hold of x: k 2^(e - 6) with whole k, at most 127, 2^e the power of two in a block's largest magnitude."""
    k = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -k % 32)).unflatten(-1, (-1, 32))
    e = (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 1).clamp_min(-120)
    code = torch.round(torch.ldexp(b, 6 - e)).clamp(-127, 127)
    return torch.ldexp(code, e - 6).flatten(-2)[..., :k]


def _act(name, a):
    """act(a) and its derivative."""
    if name == "gelu":
        phi = 0.5 * torch.erfc(-a * 0.5**0.5)
        return a * phi, phi + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5
    if name == "silu":
        s = 1 / (1 + torch.exp(-a))
        return a * s, s * (1 + a * (1 - s))
    c = 2 * (2 / math.pi) ** 0.5
    s = 1 / (1 + torch.exp(-c * (a + 0.044715 * a * a * a)))
    return a * s, s + a * s * (1 - s) * c * (1 + 3 * 0.044715 * a * a)


def _ffn_plain(s):
    dt = s["x"].dtype
    x, w1, w3, w2 = (s[k].float() for k in ("x", "w1", "w3", "w2"))
    a, b = x @ w1.t(), x @ w3.t()
    y = ((_act(s["act"], a)[0] * b) @ w2.t()).to(dt)
    if not s["grad"]:
        return y
    if s["checkpoint"] == "mx8":
        x, a, b = _held(x), _held(a), _held(b)
    dy = s["dy"].float()
    dh = dy @ w2
    g, dg = _act(s["act"], a)
    da, db = dh * b * dg, dh * g
    return {"y": y, "dx": (da @ w1 + db @ w3).to(dt), "dw1": (da.t() @ x).to(dt), "dw3": (db.t() @ x).to(dt),
            "dw2": (dy.t() @ (g * b)).to(dt)}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    import autoparallel_b200.ops as K

    if s["kind"] == "save":
        codes, scales = K.mx8_quantize(s["x"])
        return K.mx8_dequantize(codes, scales, s["x"].dtype)
    if s["kind"] == "norm8":
        y, h, q, scale = K.add_rms_norm_fp8(s["x"], s["residual"], s["w"], EPS, keep=s["keep"])
        out = {"h": h, "q": q, "scale": scale}
        return {**out, "y": y} if s["keep"] else out
    if s["kind"] == "norm":
        if not s["grad"]:
            y, h = K.add_rms_norm(s["x"], s["residual"], s["w"], EPS)
            return {"y": y, "h": h}
        leaves = [s[k].detach().requires_grad_() for k in ("x", "residual", "w")]
        y, h = K.add_rms_norm(*leaves, EPS)
        dx, dr, dw = torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dr, "dw": dw}
    leaves = [s[k] for k in ("x", "w1", "w3", "w2")]
    if not s["grad"]:
        return K.gated_ffn(*leaves, act=s["act"], checkpoint=s["checkpoint"])
    leaves = [t.detach().requires_grad_() for t in leaves]
    y = K.gated_ffn(*leaves, act=s["act"], checkpoint=s["checkpoint"])
    dx, dw1, dw3, dw2 = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), "dx": dx, "dw1": dw1, "dw3": dw3, "dw2": dw2}


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "save":
        return _held(state["x"]).to(state["x"].dtype)
    return _ffn_plain(state) if state["kind"] == "ffn" else _norm_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    m, d = case["rows"], case["d"]
    n = m * d
    if case["kind"] == "norm":
        return {"bytes": (7 if case["grad"] else 4) * n * b + d * b, "flops": (18 if case["grad"] else 6) * n}
    if case["kind"] == "norm8":
        return {"bytes": (4 if case["keep"] else 3) * n * b + n + 4 * m + d * b, "flops": 8 * n}
    if case["kind"] == "save":
        return {"bytes": 2 * n * b, "flops": 4 * n}
    w = 3 * d * case["hidden"]
    return {"bytes": (2 if case["grad"] else 1) * b * (2 * n + w), "flops": (6 if case["grad"] else 2) * m * w}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_held(x):
    k = x.shape[-1]
    out = torch.empty_like(x)
    for j in range(0, k, 32):
        block = x[..., j : j + 32]
        top = block.abs().amax(-1, keepdim=True).clamp_min(2.0**-120)
        unit = torch.exp2(torch.frexp(top).exponent.double() - 7)
        out[..., j : j + 32] = torch.clamp(torch.round(block / unit), -127, 127) * unit
    return out


def _exact_e4m3(v):
    """Nearest e4m3 number, ties to even; |v| <= 448."""
    unit = torch.exp2(torch.clamp(torch.frexp(v).exponent.double() - 4, min=-9.0))
    return torch.round(v / unit) * unit


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "save":
        return _exact_held(x)
    if case["kind"] in ("norm", "norm8"):
        # (the sum of two values of 8 or 24 bits, rounded once, is what h is defined as)
        h = (x + s["residual"].double()).to(s["x"].dtype)
        hd = h.double().requires_grad_()
        w = s["w"].double().requires_grad_()
        y = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + EPS) * w
        if case["kind"] == "norm8":
            v = y.detach()
            top = v.abs().amax(-1, keepdim=True)
            scale = torch.where(top < 2.0**-100, torch.ones_like(top), top / 448)
            out = {"h": h.double(), "q": _exact_e4m3(v / scale), "scale": scale}
            return {**out, "y": v} if case["keep"] else out
        if not case["grad"]:
            return {"y": y.detach(), "h": h.double()}
        dx, dw = torch.autograd.grad((y, hd * 1), (hd, w), (s["dy"].double(), s["dh"].double()))
        return {"y": y.detach(), "h": h.double(), "dx": dx, "dresidual": dx, "dw": dw}
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
    w1, w3, w2 = (s[k].double() for k in ("w1", "w3", "w2"))
    a, b = torch.einsum("md,hd->mh", x, w1), torch.einsum("md,hd->mh", x, w3)
    y = torch.einsum("mh,dh->md", act(a) * b, w2)
    if not case["grad"]:
        return y
    if case["checkpoint"] == "mx8":
        x, a, b = _exact_held(x), _exact_held(a), _exact_held(b)
    dy = s["dy"].double()
    a.requires_grad_()
    b.requires_grad_()
    h = act(a) * b
    da, db = torch.autograd.grad(h, (a, b), torch.einsum("md,dh->mh", dy, w2))
    return {"y": y, "dx": torch.einsum("mh,hd->md", da, w1) + torch.einsum("mh,hd->md", db, w3), "dw1": torch.einsum("mh,md->hd", da, x),
            "dw3": torch.einsum("mh,md->hd", db, x), "dw2": torch.einsum("md,mh->dh", dy, h.detach())}
