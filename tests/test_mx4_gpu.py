"""The MXFP4 kernels: conversions bit by bit against the formulas of ops/mx4_ops.py, products and gradients against 64 bits."""
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
    yield cuda_impl
    cuda_impl.check_status()


def ref(name, *args):
    from autoparallel_b200.ops import reference_impls

    return reference_impls[name](*[a.cpu() if isinstance(a, torch.Tensor) else a for a in args])


def randn(*shape, seed=0, dtype=F32):
    g = torch.Generator("cuda").manual_seed(seed)
    rows = torch.exp(2 * torch.randn(shape[:-1] + (1,), device="cuda", generator=g))
    return (torch.randn(shape, device="cuda", generator=g) * rows).to(dtype)


def check_conversions(x):
    """Codes, scales, values and rounding along both dims of ``x`` [R, K] or [E, R, K], whatever its strides."""
    codes, scales = K.mx4_quantize(x)
    rc, rs = ref("mx4_quantize", x)
    assert torch.equal(codes.cpu(), rc) and torch.equal(scales.cpu(), rs)
    for dtype in (BF16, F32):
        y = K.mx4_dequantize(codes, scales, x.shape[-1], dtype)
        assert y.is_contiguous() and torch.equal(y.cpu().nan_to_num(123.0),
                                                 ref("mx4_dequantize", rc, rs, x.shape[-1], dtype).nan_to_num(123.0))
    for dim in (-1, -2):
        y = K.mx4_round(x, dim)
        assert y.dtype == x.dtype and torch.equal(y.cpu().nan_to_num(123.0), ref("mx4_round", x, dim).nan_to_num(123.0))


@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (1, 32), (3, 33), (127, 128), (128, 129), (129, 127), (300, 1000), (64, 4096),
                                   (1, 8192),
                                   (2, 100, 72), (5, 130, 264), (3, 1, 40)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_conversions(shape, dtype):
    x = randn(*shape, dtype=dtype)
    check_conversions(x)
    check_conversions(x.transpose(-1, -2))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_conversions_of_views(dtype):
    base = randn(4, 140, 168, dtype=dtype)
    for x in (base[0, 3:, 5:], base[1, :, :96], base[:, ::2, :64], base[:, 1:130, 8:], base[::2], base[2].t()[7:, 4:], base[:, :, ::2],
              base.permute(1, 0, 2), base.permute(2, 0, 1), base[0].expand(3, 140, 168), base[0, :1].expand(140, 168),
              base[0, :, :1].expand(140, 168),
              base.view(-1)[1:1 + 64 * 96].view(64, 96), base.view(-1)[4:4 + 64 * 96].view(64, 96)):
        check_conversions(x)


def test_special_values():
    for dtype in (BF16, F32):
        x = randn(40, 96, dtype=dtype)
        x[0, 5], x[1, 40], x[2, 95], x[3, 0] = torch.inf, -torch.inf, torch.nan, -torch.nan
        x[4], x[5] = 0.0, -0.0
        x[6, :32] = torch.finfo(dtype).max
        x[7] = x[7] * 2.0**-126                  # denormals
        x[8, :32] = 2.0**-127
        x[9, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.9],
                                 device="cuda")
        x[9, 16:32] = 0
        check_conversions(x)
        check_conversions(x.t().contiguous().t())


def check_product(x, w, y, out_dtype):
    """``y`` against the exact product of the rounded operands: K additions in fp32, then the result's type."""
    xq, wq = K.mx4_round(x).double(), K.mx4_round(w).double()
    want = xq @ wq.transpose(-1, -2)
    bound = (xq.abs() @ wq.abs().transpose(-1, -2)) * (x.shape[-1] * 2.0**-24) + 1e-300
    if out_dtype == BF16:
        bound = bound + want.abs() * 2.0**-8
    assert y.dtype == out_dtype and y.shape == want.shape
    assert ((y.double() - want).abs() <= bound).all(), ((y.double() - want).abs() / bound).max().item()


PRODUCTS = [
    # (experts, M, N, K): one of every kind of tile and tail
    (0, 1, 1, 1), (0, 1, 128, 32), (0, 5, 7, 33), (0, 32, 129, 2080), (0, 33, 128, 256), (0, 128, 128, 64), (0, 128, 256, 512),
    (0, 129, 257, 96),
    (0, 300, 520, 1000), (0, 257, 132, 512), (0, 513, 392, 300), (0, 700, 1000, 777), (0, 999, 1408, 2048), (0, 2048, 2048, 1024),
    (0, 3000, 1160, 160),
    (0, 8, 20000, 4500), (0, 1, 20000, 8192), (0, 100, 40000, 600),
    (3, 130, 264, 160), (2, 257, 129, 2080), (4, 5, 264, 163), (64, 16, 1408, 256), (64, 3, 300, 1056), (5, 1280, 704, 512),
    (300, 1, 128, 64),
]


@pytest.mark.parametrize("E,M,N,k", PRODUCTS)
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_products(E, M, N, k, out_dtype):
    lead = (E,) if E else ()
    x, w = randn(*lead, M, k, seed=1), randn(*lead, N, k, seed=2)
    a, b = K.mx4_quantize(x), K.mx4_quantize(w)
    check_product(x, w, K.mx4_mm(*a, *b, out_dtype=out_dtype), out_dtype)
    check_product(x, w, K.mx4_linear(x, *b, out_dtype=out_dtype), out_dtype)
    if M * N < 1 << 20:
        check_product(x, w, K.mx4_matmul(x, w, out_dtype=out_dtype), out_dtype)
        xb = x.to(BF16)
        check_product(xb, w, K.mx4_linear(xb, *b, out_dtype=out_dtype), out_dtype)
        wt = w.transpose(-1, -2).contiguous()
        check_product(xb, w, K.mx4_matmul(xb, wt, trans_b=False, out_dtype=out_dtype), out_dtype)


@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("E,M,N,k", [(0, 1, 1, 1), (0, 200, 300, 1000), (2, 257, 129, 2080), (0, 600, 640, 512), (3, 100, 1000, 333),
                                     (2, 260, 1408, 1280),
                                     (0, 700, 2064, 300), (0, 256, 6000, 1024), (9, 700, 1760, 1100), (64, 300, 1152, 640),
                                     (2, 260, 1407, 300), (3, 131, 390, 256), (0, 513, 131, 512), (5, 97, 641, 96), (0, 2050, 66, 64)])
def test_every_tile_shape(kernels, form, E, M, N, k):
    lead = (E,) if E else ()
    x, w = randn(*lead, M, k, seed=3), randn(*lead, N, k, seed=4)
    a, b = K.mx4_quantize(x), K.mx4_quantize(w)
    for fp32 in (True, False):
        check_product(x, w, kernels.extension().mx4_mm(*a, *b, fp32, form), F32 if fp32 else BF16)


@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_rows(M, dtype):
    """Rounded in the product's launch or before it, with one slice of K and with several, rounds of the ring, and rows that are no
    whole vectors."""
    for N, k in ((256, 64), (4096, 4096), (300, 1003), (40000, 4096), (2000, 14336)):
        base = randn(M, k + 3, seed=M, dtype=dtype)
        w = randn(N, k, seed=5, dtype=BF16)
        b = K.mx4_quantize(w)
        for x in (base[:, :k].contiguous(), base[:, :k], base[:, 3:]):
            y = K.mx4_linear(x, *b, out_dtype=F32)
            check_product(x, w, y, F32)
            assert torch.equal(y, K.mx4_linear(x, *b, out_dtype=F32))
    x = randn(6, M, 160, seed=6, dtype=dtype)
    for view in (x, x[::2], x[:, :, :96], x.transpose(0, 1).contiguous().transpose(0, 1)):
        w = randn(view.shape[0], 200, view.shape[2], seed=7)
        check_product(view, w, K.mx4_linear(view, *K.mx4_quantize(w), out_dtype=F32), F32)


@pytest.mark.parametrize("M", [1, 3, 4, 8, 16, 32])
@pytest.mark.parametrize("E,N,k", [(0, 80000, 300), (0, 120000, 64), (64, 1408, 1100), (700, 128, 520), (5, 20010, 96), (300, 260, 4000)])
def test_few_rows_of_many_tiles(M, E, N, k):
    """More tiles than CTAs at once: tiles of one k-block, of fewer than a ring has slots, of more; rows that several matrices have."""
    lead = (E,) if E else ()
    x, w = randn(*lead, M, k, seed=M), randn(*lead, N, k, seed=5)
    b = K.mx4_quantize(w)
    for dtype in (BF16, F32):
        y = K.mx4_linear(x.to(dtype), *b, out_dtype=F32)
        check_product(x.to(dtype), w, y, F32)
        assert torch.equal(y, K.mx4_linear(x.to(dtype), *b, out_dtype=F32))
    check_product(x, w, K.mx4_mm(*K.mx4_quantize(x), *b), BF16)


def test_shapes_of_x():
    w = randn(48, 64, seed=1)
    b = K.mx4_quantize(w)
    x = randn(2, 3, 5, 64, seed=2)
    y = K.mx4_linear(x, *b)
    assert y.shape == (2, 3, 5, 48) and torch.equal(y.view(30, 48), K.mx4_linear(x.view(30, 64), *b))
    assert torch.equal(K.mx4_linear(x[0, 0, 0], *b), y[0, 0, 0])
    assert torch.equal(K.mx4_matmul(x.transpose(0, 1), w), y.transpose(0, 1))
    for shape in ((0, 64), (2, 0, 64)):
        assert K.mx4_linear(torch.zeros(shape, device="cuda"), *b).shape == (*shape[:-1], 48)
    assert K.mx4_linear(x[0, 0], *K.mx4_quantize(w[:0])).shape == (5, 0)
    assert (K.mx4_matmul(x[0, 0, :, :0], w[:, :0]) == 0).all()
    assert K.mx4_quantize(w[:0])[0].shape == (0, 32) and K.mx4_round(w[:0]).shape == (0, 64)


def test_broken_blocks_stay_in_their_rows_and_columns():
    for M, N, k in ((4, 300, 512), (20, 300, 512), (300, 400, 640)):
        x, w = randn(M, k, seed=1), randn(N, k, seed=2)
        x[1, 100], w[7, 33], w[N - 1, k - 1] = torch.nan, torch.inf, torch.nan
        y = K.mx4_matmul(x, w)
        bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
        bad[1], bad[:, 7], bad[:, N - 1] = True, True, True
        assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("lead,m,n,k,trans_b", [((), 64, 96, 128, True), ((), 37, 40, 72, False), ((), 37, 41, 75, True),
                                                ((), 300, 264, 520, False),
                                                ((3,), 40, 64, 96, False), ((2,), 33, 50, 77, True), ((2, 5), 8, 24, 64, True)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients(lead, m, n, k, trans_b, dtype):
    grouped = len(lead) == 1
    wl = lead if grouped else ()
    x, dy = randn(*lead, m, k, seed=1, dtype=dtype).requires_grad_(), torch.randn(*lead, m, n, device="cuda").to(dtype)
    w = randn(*wl, *((n, k) if trans_b else (k, n)), seed=2, dtype=dtype).requires_grad_()
    dx, dw = torch.autograd.grad(K.mx4_matmul(x, w, trans_b=trans_b), (x, w), dy)
    xq, wq = K.mx4_round(x.detach()).double(), K.mx4_round(w.detach(), -1 if trans_b else -2).double()
    wq = wq if trans_b else wq.transpose(-1, -2)
    d = dy.double()
    if not grouped:
        xq, d2 = xq.reshape(-1, k), d.reshape(-1, n)
    else:
        d2 = d
    want_dx, want_dw = d @ wq, d2.transpose(-1, -2) @ xq
    want_dw = want_dw if trans_b else want_dw.transpose(-1, -2)
    tol = 2.0**-7 if dtype == BF16 else 1e-4

    def near(a, b):
        return ((a.double() - b).norm() / b.norm()).item() <= tol and a.shape == b.shape and a.dtype == dtype

    assert near(dx, want_dx) and near(dw, want_dw)
    # one operand alone
    (only,) = torch.autograd.grad(K.mx4_matmul(x, w.detach(), trans_b=trans_b), x, dy)
    assert torch.equal(only, dx)
    (only,) = torch.autograd.grad(K.mx4_matmul(x.detach(), w, trans_b=trans_b), w, dy)
    assert torch.equal(only, dw)
    b = K.mx4_quantize(w.detach() if trans_b else w.detach().transpose(-1, -2))
    (dl,) = torch.autograd.grad(K.mx4_linear(x, *b), x, dy)
    assert near(dl, want_dx)
    (dr,) = torch.autograd.grad(K.mx4_round(x), x, torch.ones_like(x))
    assert (dr == 1).all()


@pytest.mark.parametrize("E,M,N,k", [(0, 1, 8, 16), (0, 5, 64, 256), (0, 128, 128, 272), (0, 129, 200, 512), (0, 256, 72, 1000),
                                     (0, 300, 1408, 2048), (0, 2000, 520, 640),
                                     (3, 40, 136, 96), (64, 160, 264, 512), (2, 513, 640, 1040)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_products_with_the_values_of_codes(kernels, E, M, N, k, out_dtype):
    """The kernel that turns codes to values on the way (whatever the size), and the operator, against 64 bits; the values themselves bit by
    bit."""
    lead = (E,) if E else ()
    a, w = torch.randn(*lead, M, N, device="cuda", dtype=BF16), randn(*lead, N, k, seed=2)
    if M == 5:
        w[3, :32], w[4, :40] = torch.finfo(F32).max, 2.0**-127  # the ends of the scales
    codes, scales = K.mx4_quantize(w)
    values = K.mx4_dequantize(codes, scales, k, F32).double()
    want = a.double() @ values
    bound = (a.double().abs() @ values.abs()) * (N * 2.0**-24) + (want.abs() * 2.0**-8 if out_dtype == BF16 else 0) + 1e-300
    for c in (kernels.extension().mx4_mm_values(a, codes, scales, k, out_dtype == F32, True),
              K.mx4_mm_values(a, codes, scales, k, out_dtype)):
        near = ((c.double() - want).abs() <= bound) | (c == want.to(F32).to(out_dtype))  # (or both beyond the type's range)
        assert c.shape == want.shape and c.dtype == out_dtype and near.all()
    n = min(M, N)
    eye = torch.eye(N, device="cuda", dtype=BF16)[:n].expand(*lead, n, N).contiguous()
    c = kernels.extension().mx4_mm_values(eye, codes, scales, k, True, True)
    assert torch.equal(c.double(), values[..., :n, :])
    before = K.mx4_mm_values(a, codes, scales, k, F32)
    w[..., N - 1, k - 1] = torch.nan
    c, first = K.mx4_mm_values(a, *K.mx4_quantize(w), k, F32), (k - 1) // 32 * 32
    assert c[..., first:].isnan().all() and torch.equal(c[..., :first], before[..., :first])


def test_an_installed_function_is_what_runs():
    from autoparallel_b200.ops import library, register_cuda_impl

    own, calls = library._cuda_table["mx4_matmul"], []
    x, w = randn(64, 64).requires_grad_(), randn(32, 64, seed=1).requires_grad_()
    want = K.mx4_matmul(x, w)
    grads = torch.autograd.grad(want, (x, w), torch.ones_like(want))
    register_cuda_impl("mx4_matmul", lambda *a: calls.append(1) or own(*a))
    try:
        y = K.mx4_matmul(x, w)
        again = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    finally:
        register_cuda_impl("mx4_matmul", own)
    assert calls == [1] and torch.equal(y, want) and all(torch.allclose(a, b) for a, b in zip(grads, again, strict=True))


def test_native_entries_answer_as_the_python_ones():
    from autoparallel_b200.ops import cuda_impl, library

    x, w = randn(40, 96), randn(24, 96, seed=1)
    a, b = K.mx4_quantize(x), K.mx4_quantize(w)
    r = torch.randn(6, 16, device="cuda")
    route = library.ops.moe_route(r, None, 4, False, 1, 1, True, 1.0)
    for name, args in (("mx4_quantize", (x,)), ("mx4_dequantize", (*a, 96, BF16)), ("mx4_round", (x, -2)), ("mx4_mm", (*a, *b, F32)),
                       ("mx4_mm_values", (x.bfloat16()[:1].expand(160, 40, 96), *K.mx4_quantize(randn(160, 96, 64, seed=2)), 64, BF16)),
                       ("mx4_linear", (x, *b, BF16)), ("mx4_linear", (x[:3], *b, BF16)), ("mx4_matmul", (x, w, True, F32)),
                       ("moe_route", (r, None, 4, False, 1, 1, True, 1.0)), ("moe_route_bwd", (route[0], r, route[1], False, True, 1.0))):
        results = []
        for fn in (getattr(library.ops, name), library._cuda_table[name]):
            before = cuda_impl.launch_count
            out = fn(*args)
            results.append((out if isinstance(out, tuple) else (out,), cuda_impl.launch_count - before))
        assert results[0][1] == results[1][1] > 0, name
        assert all(torch.equal(p, q) for p, q in zip(results[0][0], results[1][0], strict=True)), name


def test_another_stream_and_a_graph():
    x, w = randn(256, 512, dtype=BF16), randn(384, 512, seed=1, dtype=BF16)
    b = K.mx4_quantize(w)
    want, want_few = K.mx4_linear(x, *b), K.mx4_linear(x[:3], *b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, few = K.mx4_linear(x * 1, *b), K.mx4_linear(x[:3] * 1, *b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want) and torch.equal(few, want_few)
    g = torch.cuda.CUDAGraph()
    held = x.clone()
    with torch.cuda.graph(g):
        y, few = K.mx4_linear(held, *b), K.mx4_linear(held[:3], *b)
    held.copy_(-x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, -want) and torch.equal(few, -want_few)


def test_long_stack_passes_32_bit_offsets():
    """More than 2^31 values in a stack: the last matrices are read and written where they lie."""
    E, R, k = 33, 8192, 8192
    x = torch.zeros(E, R, k, device="cuda", dtype=BF16)
    x[-1] = randn(R, k, dtype=BF16)
    codes, scales = K.mx4_quantize(x)
    c, s = K.mx4_quantize(x[-1])
    assert torch.equal(codes[-1], c) and torch.equal(scales[-1], s) and (codes[:-1] == 0).all()
    y = K.mx4_dequantize(codes, scales)
    assert torch.equal(y[-1], K.mx4_dequantize(c, s)) and (y[:-1] == 0).all()
    w = randn(128, k, seed=1, dtype=BF16)
    wc, ws = K.mx4_quantize(w.expand(E, 128, k))
    z = K.mx4_linear(x, wc, ws)
    assert torch.equal(z[-1], K.mx4_linear(x[-1], *K.mx4_quantize(w))) and (z[:-1] == 0).all()


def test_refusals_of_the_operators():
    apb = torch.ops.apb200
    x, w = randn(8, 64), randn(8, 64, seed=1)
    a, b = K.mx4_quantize(x), K.mx4_quantize(w)
    for call in (
        lambda: apb.mx4_quantize(x.half()), lambda: apb.mx4_quantize(x[0]), lambda: apb.mx4_dequantize(*a, 65, F32),
        lambda: apb.mx4_dequantize(*a, 64, torch.half),
        lambda: apb.mx4_dequantize(a[0], a[1][..., :256], 64, F32), lambda: apb.mx4_dequantize(a[0], a[1].cpu(), 64, F32),
        lambda: apb.mx4_round(x, 0),
        lambda: apb.mx4_mm(*a, *K.mx4_quantize(w[:, :32]), F32), lambda: apb.mx4_mm(*a, b[0][None], b[1][None], F32),
        lambda: apb.mx4_mm(*a, *b, torch.half),
        lambda: apb.mx4_linear(x[:, :32], *b, F32), lambda: apb.mx4_linear(x.double(), *b, F32),
        lambda: apb.mx4_linear(x, b[0].cpu(), b[1].cpu(), F32),
        lambda: apb.mx4_matmul(x, w, False, F32), lambda: apb.mx4_matmul(x, w[:, :32], True, F32),
    ):
        with pytest.raises(RuntimeError):
            call()


def test_c_entries_refuse_what_they_cannot_take():
    from autoparallel_b200.ops import build

    so = ctypes.CDLL(build.so_path())
    i64, ptr = ctypes.c_longlong, ctypes.c_void_p
    x, out = torch.zeros(4, 64, device="cuda"), torch.zeros(1 << 16, device="cuda", dtype=torch.uint8)
    p = out.data_ptr()
    quantize, mm, rows = so.apb_mx4_quantize, so.apb_gemm_mx4, so.apb_gemm_mx4_rows
    q = lambda codes, scales, K_=64: quantize(ptr(x.data_ptr()), ptr(codes), ptr(scales), i64(1), i64(4), i64(K_), i64(0), i64(64), 0, 0,
                                              ptr(0))  # noqa: E731
    assert q(p, p + 4096) == 0 and q(p + 8, p + 4096) == 3 and q(p, p + 4) == 3 and q(p, p + 4096, -1) == 3
    status = torch.zeros(4, dtype=torch.int32, device="cuda")

    def product(f, tail, a=p, c=p + 32768, kp=64, n=8):
        return f(ptr(a), ptr(p + 8192), ptr(p + 16384), ptr(p + 20480), ptr(c), i64(1), i64(4), i64(n), i64(kp), *tail)

    tail = (1, -1, ptr(status.data_ptr()), 148, ptr(0))
    assert product(mm, tail) == 0 and product(mm, tail, a=p + 4) == 3 and product(mm, tail, c=p + 32776) == 3
    assert product(mm, tail, kp=48) == 3
    assert product(mm, tail, n=-1) == 3
    tail = (i64(0), i64(0), 2, 1, 0, ptr(status.data_ptr()), 148, ptr(0))
    assert product(rows, tail) == 0 and product(rows, tail, a=p + 4) == 3
    assert product(rows, (i64(0), i64(0), 2, 1, 3, ptr(status.data_ptr()), 148, ptr(0))) == 3
    torch.cuda.synchronize()

@pytest.mark.parametrize("shape", [(0,), (4, 0), (2, 5, 0), (2, 3, 40, 0)])
def test_contractions_of_nothing_are_zero(shape):
    """Whatever the dims of x, and in memory that held something else."""
    w = torch.zeros(48, 0, device="cuda", requires_grad=True)
    b = K.mx4_quantize(w.detach())
    for dtype in (BF16, F32):
        held = torch.full((*shape[:-1], 48), 7.0, device="cuda", dtype=dtype)
        del held
        x = torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True)
        y = K.mx4_linear(x, *b)
        assert y.shape == (*shape[:-1], 48) and y.dtype == dtype and (y == 0).all()
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert dx.shape == shape
        y = K.mx4_matmul(x, w)
        assert y.shape == (*shape[:-1], 48) and (y == 0).all()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert dx.shape == shape and dw.shape == w.shape
        assert K.mx4_mm_values(y.detach(), *b, 0).shape == shape


@pytest.mark.parametrize("lead,m,n,k", [((), 5, 0, 64), ((), 0, 48, 64), ((3,), 5, 0, 64), ((3,), 5, 48, 0), ((3,), 0, 48, 64),
                                        ((0,), 5, 48, 64), ((2, 3), 5, 0, 64), ((), 5, 0, 0)])
@pytest.mark.parametrize("trans_b", [True, False])
def test_matrices_of_nothing(lead, m, n, k, trans_b):
    """Products and gradients without rows, columns, experts or a contraction."""
    wl = lead if len(lead) == 1 else ()
    for dtype in (BF16, F32):
        x = torch.randn(*lead, m, k, device="cuda").to(dtype).requires_grad_()
        w = torch.randn(*wl, *((n, k) if trans_b else (k, n)), device="cuda").to(dtype).requires_grad_()
        y = K.mx4_matmul(x, w, trans_b=trans_b)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        codes, scales = K.mx4_quantize(w.detach() if trans_b else w.detach().transpose(-1, -2))
        z = K.mx4_linear(x, codes, scales)
        (dz,) = torch.autograd.grad(z, x, torch.ones_like(z))
        v = K.mx4_mm_values(y.detach(), codes, scales, k)
        assert y.shape == z.shape == (*lead, m, n) and dx.shape == dz.shape == v.shape == x.shape and dw.shape == w.shape
        assert all((t == 0).all() for t in (y, z, dx, dz, dw, v))


@pytest.mark.parametrize("lead,m,n,k", [((), 64, 96, 128), ((), 37, 40, 72), ((), 37, 41, 75), ((3,), 40, 64, 96), ((2,), 33, 50, 77),
                                        ((2, 5), 8, 24, 64), ((160,), 20, 96, 256)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_products_with_values(lead, m, n, k, dtype):
    """a . values has the gradient dc . values^T; so has the gradient of mx4_linear, which is such a product."""
    wl = lead if len(lead) == 1 else ()
    codes, scales = K.mx4_quantize(randn(*wl, n, k, seed=2, dtype=dtype))
    values = K.mx4_dequantize(codes, scales, k, F32).double().transpose(-1, -2)
    a = torch.randn(*lead, m, n, device="cuda").to(dtype).requires_grad_()
    dc = torch.randn(*lead, m, k, device="cuda").to(dtype)
    want = dc.double() @ values
    tol = 2.0**-7 if dtype == BF16 else 1e-4  # (the type of the result, of the norm)

    def near(g):
        return g.dtype == dtype and g.shape == a.shape and ((g.double() - want).norm() / want.norm()).item() <= tol

    (da,) = torch.autograd.grad(K.mx4_mm_values(a, codes, scales, k), a, dc)
    assert near(da)
    x = torch.randn(*lead, m, k, device="cuda").to(dtype).requires_grad_()
    (dx,) = torch.autograd.grad(K.mx4_linear(x, codes, scales), x, a, create_graph=True)
    (da,) = torch.autograd.grad(dx, a, dc)
    assert near(da)
    with torch.no_grad():
        assert not K.mx4_mm_values(a, codes, scales, k).requires_grad


@pytest.mark.parametrize("wrt", ["x", "w", "dy"])
def test_second_derivatives_of_matmul_are_refused(wrt):
    """The operands are kept in 4 bits alone, so the gradients cannot be differentiated: they say so where they are, and are themselves as
    ever."""
    x, w = randn(40, 64).requires_grad_(), randn(32, 64, seed=1).requires_grad_()
    dy = torch.randn(40, 32, device="cuda").requires_grad_()
    y = K.mx4_matmul(x, w)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and not want[0].requires_grad
    for g in (dx, dw):
        with pytest.raises(RuntimeError, match="mx4_matmul: no second derivatives"):
            torch.autograd.grad((g * g).sum() + w.sum() + x.sum() + dy.sum(), {"x": x, "w": w, "dy": dy}[wrt], retain_graph=True)


@pytest.mark.parametrize("M", [1, 3, 16, 17, 32])
def test_every_number_of_slices(M):
    """The kernel for few rows with the slices of K that it is told to take, one to four CTAs a cluster, from codes and from values; more
    are refused."""
    from autoparallel_b200.ops import build, cuda_impl

    rows, i64, ptr = ctypes.CDLL(build.so_path()).apb_gemm_mx4_rows, ctypes.c_longlong, ctypes.c_void_p
    N, k = 300, 1100
    x, w = randn(M, k, seed=1), randn(N, k, seed=2)
    (a, sa), (b, sb) = K.mx4_quantize(x), K.mx4_quantize(w)
    status = cuda_impl.status_buffer(x.device)
    torch.cuda.synchronize()

    def call(A, SA, kind, K_, slices, y):
        return rows(*[ptr(t.data_ptr()) for t in (A, SA, b, sb, y)], i64(1), i64(M), i64(N), i64(K_), i64(0), i64(k), kind, 1, slices,
                    ptr(status.data_ptr()), 148, ptr(0))

    for slices in (1, 2, 4):
        y = torch.zeros(M, N, device="cuda")
        assert call(a, sa, 2, 2 * a.shape[1], slices, y) == 0
        torch.cuda.synchronize()
        check_product(x, w, y, F32)
        for kind, v in ((0, x), (1, x.to(BF16))):
            y = torch.zeros(M, N, device="cuda")
            assert call(v, v, kind, k, slices, y) == (0 if M <= 16 else 3)
            torch.cuda.synchronize()
            check_product(v, w, y, F32) if M <= 16 else None
    assert call(a, sa, 2, 2 * a.shape[1], 8, y) == 3


@pytest.mark.parametrize("E,M,N,k,launches", [(0, 4, 4096, 14336, 1), (0, 5, 4096, 4096, 1), (0, 8, 4096, 4096, 1), (0, 9, 4096, 4096, 2),
                                              (0, 8, 4096, 6144, 2), (0, 8, 14336, 2048, 1), (0, 8, 14336, 4096, 2), (8, 8, 4096, 1024, 1),
                                              (8, 8, 4096, 2048, 2), (64, 8, 1408, 1024, 2), (64, 4, 1408, 2048, 1)])
def test_where_few_rows_are_rounded(kernels, E, M, N, k, launches):
    """Inside the product's launch, or before it where a CTA would have many blocks of all rows to round; the same bits either way."""
    lead = (E,) if E else ()
    x, b = randn(*lead, M, k, seed=1, dtype=BF16), K.mx4_quantize(randn(*lead, N, k, seed=2, dtype=BF16))
    before = kernels.launch_count
    y = K.mx4_linear(x, *b)
    assert kernels.launch_count - before == launches
    assert torch.equal(y, K.mx4_mm(*K.mx4_quantize(x), *b))
