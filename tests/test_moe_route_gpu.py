"""The routing kernels against the formula of ops/moe_ops.py, evaluated by torch on the same device, and in 64 bits."""
import ctypes

import pytest
import torch

import autoparallel_b200.ops as K

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def kernels():
    from autoparallel_b200.ops import cuda_impl

    cuda_impl.ensure_loaded()
    yield
    cuda_impl.check_status()


def formula(logits, bias, k, score, groups, top_groups, renormalize, scale):
    from autoparallel_b200.ops import reference_impls

    return reference_impls["moe_route"](logits, bias, k, score == "sigmoid", groups, top_groups, renormalize, scale)


def exact_weights(logits, idx, score, renormalize, scale):
    x = logits.double()
    s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
    if score == "softmax" and renormalize:
        return scale * torch.softmax(x.gather(-1, idx), -1)
    p = s.gather(-1, idx)
    return scale * (p / p.sum(-1, keepdim=True) if renormalize else p)


def exact_gradient(logits, idx, dw, score, renormalize, scale):
    z = logits.double().requires_grad_()
    return torch.autograd.grad(exact_weights(z, idx, score, renormalize, scale), z, dw.double())[0]


def check(x, k, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    xg = x.detach().requires_grad_()
    w, idx = K.moe_route(xg, k, score=score, bias=bias, num_groups=groups, top_groups=top_groups, renormalize=renormalize, scale=scale)
    rw, ridx = formula(x, bias, k, score, groups, top_groups, renormalize, scale)
    assert torch.equal(idx, ridx)
    # sums of at most 1024 scores in fp32, an exponential to 2 units in the last place, one division
    assert torch.allclose(w.double(), exact_weights(x, idx, score, renormalize, scale), rtol=2e-5, atol=1e-12)
    dw = torch.randn(w.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    (dx,) = torch.autograd.grad(w, xg, dw)
    want = exact_gradient(x, idx, dw, score, renormalize, scale)
    tol = 2.0**-8 if x.dtype == BF16 else 1e-4  # (the result's type; in fp32 the differences of products that nearly cancel)
    assert dx.dtype == x.dtype and torch.allclose(dx.double(), want, rtol=tol, atol=tol * 0.02 * want.abs().max().item() + 1e-12)


def logits(T, E, dtype, seed=0, spread=1.5):
    return (spread * torch.randn(T, E, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))).to(dtype)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (3, 1), (8, 2), (31, 4), (32, 8), (33, 5), (60, 6), (64, 8), (65, 9), (128, 6),
                                 (128, 16), (130, 3),
                                 (160, 17), (256, 8), (257, 8), (512, 32), (1000, 10), (1024, 32)])
@pytest.mark.parametrize("T", [1, 2, 37, 1000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes(T, E, k, dtype):
    x = logits(T, E, dtype)
    bias = 0.001 * torch.randint(-50, 51, (E,), device="cuda").float()
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            check(x, k, score, None, renormalize=renormalize)
            check(x, k, score, bias, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("E,groups,top_groups,k", [(256, 8, 4, 8), (256, 8, 1, 8), (64, 8, 3, 6), (64, 64, 10, 8), (60, 4, 2, 5),
                                                   (160, 8, 3, 6),
                                                   (16, 4, 2, 4), (240, 5, 2, 8), (1024, 64, 4, 16), (1000, 10, 5, 32), (48, 3, 2, 8),
                                                   (40, 2, 2, 10)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups(E, groups, top_groups, k, score, dtype):
    x = logits(513, E, dtype, seed=E)
    bias = 0.001 * torch.randint(-50, 51, (E,), device="cuda").float()
    check(x, k, score, bias, groups, top_groups)
    check(x, k, score, None, groups, top_groups, renormalize=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 8])
def test_near_and_exact_ties(score, groups):
    """Values from a small set, biases a few units in the last place apart: every choice hangs on the exact order."""
    g = torch.Generator("cuda").manual_seed(3)
    x = 0.25 * torch.randint(-8, 9, (2000, 64), device="cuda", generator=g).float()
    for bias in (None, 3e-8 * torch.randint(-4, 5, (64,), device="cuda", generator=g).float(), torch.full((64,), -0.0, device="cuda")):
        check(x, 8, score, bias, groups, max(1, groups // 2))
        check(x.bfloat16(), 8, score, bias, groups, max(1, groups // 2))
    check(20 + x, 8, score, None, groups, max(1, groups // 2))  # (sigmoids that round to 1)
    check(x * 1e-7, 8, score, None, groups, max(1, groups // 2))


def test_masks_and_infinities():
    for dtype in (BF16, F32):
        x = logits(64, 64, dtype)
        x[0] = -torch.inf                       # nothing left
        x[1, 3:] = -torch.inf                   # fewer than k left
        x[2] = torch.finfo(dtype).min
        x[3, 5] = torch.finfo(dtype).min
        x[4, ::2] = -torch.inf
        x[5, 7] = torch.nan
        x[6, 9] = torch.inf
        for score in ("softmax", "sigmoid"):
            for groups in (1, 8, 16):
                for renormalize in (True, False):
                    xg = x.detach().requires_grad_()
                    w, idx = K.moe_route(xg, 8, score=score, num_groups=groups, top_groups=max(1, groups // 2), renormalize=renormalize)
                    rw, ridx = formula(x, None, 8, score, groups, max(1, groups // 2), renormalize, 1.0)
                    assert torch.equal(idx, ridx)
                    assert torch.allclose(w, rw, rtol=2e-5, atol=1e-12, equal_nan=True)
                    (dx,) = torch.autograd.grad(w, xg, torch.ones_like(w))
                    ok = torch.ones(64, dtype=torch.bool, device="cuda")
                    ok[5] = ok[6] = False
                    assert torch.isfinite(dx[ok]).all() and (dx[0] == 0).all() and (w[0] == 0).all()


def test_strides_offsets_and_leading_dims():
    base = logits(130, 200, F32)
    for x in (base[:, 3:67], base[::2, :64], base.t()[:64, :64], base[1:].reshape(-1)[1:1 + 128 * 64].view(128, 64),
              base[:, :64].reshape(2, 65, 64)):
        check(x, 8)
        check(x.bfloat16(), 8, "sigmoid", groups=4, top_groups=2)
    w, idx = K.moe_route(torch.zeros(0, 64, device="cuda"), 8)
    assert w.shape == idx.shape == (0, 8)
    xg = torch.zeros(0, 64, device="cuda", requires_grad=True)
    assert torch.autograd.grad(K.moe_route(xg, 8)[0].sum(), xg)[0].shape == (0, 64)


def test_large_batch_and_another_stream():
    x = logits(70001, 64, BF16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 1
        w, idx = K.moe_route(y, 8)
    torch.cuda.current_stream().wait_stream(s)
    rw, ridx = formula(x, None, 8, "softmax", 1, 1, True, 1.0)
    assert torch.equal(idx, ridx) and torch.allclose(w, rw, rtol=2e-5)
    w2, idx2 = K.moe_route(x, 8)
    assert torch.equal(w, w2) and torch.equal(idx, idx2)


def test_refusals_of_the_operator():
    apb, x = torch.ops.apb200, torch.zeros(4, 64, device="cuda")
    for args in ((x, None, 33, False, 1, 1, True, 1.0), (x, None, 8, False, 3, 1, True, 1.0), (x, None, 8, False, 16, 1, True, 1.0),
                 (x, torch.zeros(63, device="cuda"), 8, False, 1, 1, True, 1.0), (x, torch.zeros(64), 8, False, 1, 1, True, 1.0),
                 (x.half(), None, 8, False, 1, 1, True, 1.0), (torch.zeros(4, 1025, device="cuda"), None, 8, False, 1, 1, True, 1.0)):
        with pytest.raises(RuntimeError):
            apb.moe_route(*args)
    w, idx = K.moe_route(x, 8)
    with pytest.raises(RuntimeError):
        apb.moe_route_bwd(w[:, :4], x, idx, False, True, 1.0)
    with pytest.raises(RuntimeError):
        apb.moe_route_bwd(w, x, idx.int(), False, True, 1.0)
    # a number that names no expert has no gradient, and touches nothing
    idx[0, 0], idx[1, 0] = 64, -1
    assert torch.isfinite(apb.moe_route_bwd(w, x, idx, False, True, 1.0)).all()


def test_a_bias_that_begins_anywhere():
    """One layer's part of a flat buffer: dense, four bytes off the alignment that the kernel's 16-byte loads need."""
    g = torch.Generator("cuda").manual_seed(2)
    flat = 0.1 * torch.randn(2100, device="cuda", generator=g)
    for E in (60, 64, 256, 1024):
        for dtype in (BF16, F32):
            x = logits(300, E, dtype)
            for first in (1, 2, 3, 4):
                for score in ("softmax", "sigmoid"):
                    check(x, 5, score, flat[first : first + E])
            check(x, 5, "sigmoid", flat[: 2 * E : 2])


def test_the_c_entry_refuses_what_it_cannot_take():
    from autoparallel_b200.ops import build

    route, i64, ptr = ctypes.CDLL(build.so_path()).apb_moe_route, ctypes.c_longlong, ctypes.c_void_p
    x, bias = torch.zeros(8, 64, device="cuda"), torch.zeros(128, device="cuda")
    w, idx = torch.full((4, 8), 7.0, device="cuda"), torch.full((4, 8), -7, device="cuda")

    def call(x_bytes=0, bias_bytes=0, E=64, k=8):
        return route(ptr(x.data_ptr() + x_bytes), ptr(bias.data_ptr() + bias_bytes), ptr(w.data_ptr()), ptr(idx.data_ptr()), i64(4), E, k,
                     1, 1, 1, 1, ctypes.c_float(1.0), 0, ptr(0))

    assert call(x_bytes=4) == 3 and call(bias_bytes=4) == 3 and call(bias_bytes=8) == 3 and call(k=33) == 3 and call(E=1025) == 3
    assert (w == 7).all() and (idx == -7).all()  # nothing ran
    assert call(bias_bytes=16) == 0
    torch.cuda.synchronize()
    assert (w == 0.125).all() and (idx == torch.arange(8, device="cuda")).all()


def experts_at_random(T, E, n, g):
    """``n`` different experts of each of ``T`` tokens, in no order."""
    return torch.rand(T, E, device="cuda", generator=g).argsort(-1)[:, :n]


def same_choice(x, k, score, bias=None, groups=1, top_groups=1):
    _, idx = K.moe_route(x, k, score=score, bias=bias, num_groups=groups, top_groups=top_groups)
    wrong = (idx != formula(x, bias, k, score, groups, top_groups, True, 1.0)[1]).any(-1)
    assert not wrong.any(), f"{int(wrong.sum())} of {len(x)} tokens, first {wrong.nonzero()[0].item()}"


LAST_PLACE = [(64, 1), (64, 6), (64, 7), (64, 8), (128, 6), (256, 1), (256, 8), (256, 16), (1024, 10), (1024, 31), (60, 3)]


@pytest.mark.parametrize("E,k", LAST_PLACE)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_last_place_among_near_and_equal_values(E, k, score):
    """The last choice and the best of the rest may be equal where a third expert, with a higher number, is larger by a unit in the last
    place: several experts a few units apart contend for the last places, below others that are chosen for sure."""
    g = torch.Generator("cuda").manual_seed(E + k)
    T = 2000
    at = experts_at_random(T, E, k - 1 + 6, g)
    sure = 2 + 0.1 * torch.rand(T, k - 1, device="cuda", generator=g)
    for near in (1 + 2.0**-23 * torch.randint(0, 4, (T, 6), device="cuda", generator=g),     # fp32 neighbours
                 1 + 2.0**-20 * torch.randint(0, 3, (T, 6), device="cuda", generator=g),     # sigmoids some units apart
                 torch.full((T, 6), 1.0, device="cuda")):
        x = (torch.rand(T, E, device="cuda", generator=g) - 5).scatter_(1, at, torch.cat((sure, near.float()), 1))
        same_choice(x, k, score)
        same_choice(x, k, score, bias=3e-8 * torch.randint(-4, 5, (E,), device="cuda", generator=g).float())
        if E % 4 == 0:
            same_choice(x, k, score, groups=4, top_groups=4)
    # scores that are all but 1: different logits, the same or neighbouring sigmoids
    x = (8 + 2 * torch.randn(T, E, device="cuda", generator=g)).bfloat16()
    same_choice(x, k, score)
    same_choice(x.float(), k, score)
    same_choice(x.float() + 4, k, score)
    # few values: equal logits in most last places
    x = (0.25 * torch.randint(-8, 9, (T, E), device="cuda", generator=g)).bfloat16()
    for bias in (None, 3e-8 * torch.randint(-4, 5, (E,), device="cuda", generator=g).float()):
        same_choice(x, k, score, bias)
        same_choice(x.float(), k, score, bias)


@pytest.mark.parametrize("E,k", LAST_PLACE)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_last_place_by_hand(E, k, score):
    sure = list(range(E - k + 1, E))
    x = torch.full((4, E), -5.0, device="cuda")
    x[:, sure] = 40.0 - torch.arange(k - 1, device="cuda") / 4
    x[0, :3] = torch.tensor([12.0, 12.0, 13.0])
    x[1, :3] = torch.tensor([10.0625, 10.0625, 10.125])
    x[2, :3] = torch.tensor([1.0, 1.0, 1.0 + 2.0**-20])
    x[3, :3] = torch.tensor([1.0, 1.0, 1.0 + 2.0**-23])
    rows = 4 if score == "softmax" else 2  # (two units of a logit are less than one of a sigmoid)
    _, idx = K.moe_route(x[:rows], k, score=score)
    assert idx[:, -1].tolist() == [2] * rows and idx[:, :-1].tolist() == [sure] * rows
    _, idx = K.moe_route(x[:2].bfloat16(), k, score=score)
    assert idx[:, -1].tolist() == [2, 2]


@pytest.mark.parametrize("E,k", [(64, 1), (128, 6), (256, 8), (1024, 10)])
def test_the_last_place_at_the_ends_of_keys(E, k):
    """Keys hold the upper bits of a score.  Two scores lie within the error of a fast sigmoid to both sides of a multiple of the lower
    ones' range, and a smaller one, with a lower number, just below in the same range as the lower of the two."""
    g = torch.Generator("cuda").manual_seed(E)
    T, bits = 50000, (E - 1).bit_length()
    unit = 2.0 ** (bits - 24)  # of scores in [0.5, 1)
    at = experts_at_random(T, E, k + 2, g)
    at[:, :3] = at[:, :3].sort(-1).values
    end = (torch.randint(int(0.55 / unit), int(0.8 / unit), (T,), device="cuda", generator=g) * unit).double()
    score = torch.stack((end - 0.6 * unit, end, end), 1)
    score[:, 1:] += 4e-7 * (2 * torch.rand(T, 2, device="cuda", generator=g, dtype=torch.float64) - 1)
    x = (torch.rand(T, E, device="cuda", generator=g) - 5).scatter_(1, at, 3.0)
    x = x.scatter_(1, at[:, :3], torch.logit(score).float())
    same_choice(x, k, "sigmoid")


def test_groups_whose_two_largest_cancel():
    """The sum of two large values of unlike sign is small, but has their rounding."""
    g = torch.Generator("cuda").manual_seed(5)
    for E, groups in ((64, 8), (256, 8), (48, 3), (16, 8)):
        size = E // groups
        bias = torch.full((groups, size), -300.0, device="cuda")
        bias[:, 0], bias[:, 1] = 100.0, -100.0
        x = 0.0005 * torch.randn(100000, E, device="cuda", generator=g) - 1.5
        kept = max(1, groups // 2)
        same_choice(x, kept, "sigmoid", bias.flatten(), groups, kept)  # (the largest of every group that stays)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two devices")
def test_the_gradient_refuses_tensors_of_another_device():
    x = torch.zeros(4, 64, device="cuda:0")
    w, idx = K.moe_route(x, 8)
    for dw, i in ((w.to("cuda:1"), idx), (w, idx.to("cuda:1"))):
        with pytest.raises(RuntimeError, match="one device"):
            torch.ops.apb200.moe_route_bwd(dw, x, i, False, True, 1.0)


def test_the_gradient_refuses_tensors_of_the_host():
    x = torch.zeros(4, 64, device="cuda")
    w, idx = K.moe_route(x, 8)
    for dw, i in ((w.cpu(), idx), (w, idx.cpu())):
        with pytest.raises(RuntimeError, match="one device"):
            torch.ops.apb200.moe_route_bwd(dw, x, i, False, True, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_second_derivatives_are_refused(score):
    x, dw = logits(20, 64, F32).requires_grad_(), torch.randn(20, 8, device="cuda").requires_grad_()
    w, _ = K.moe_route(x, 8, score=score)
    (want,) = torch.autograd.grad(w, x, dw, retain_graph=True)
    (dx,) = torch.autograd.grad(w, x, dw, create_graph=True)
    assert torch.equal(dx, want) and not want.requires_grad
    for t in (x, dw):
        with pytest.raises(RuntimeError, match="moe_route: no second derivatives"):
            torch.autograd.grad((dx * dx).sum() + x.sum() + dw.sum(), t, retain_graph=True)
