// The feed-forward block's operators (ops/ffn_ops.py): checks, allocation and launches.  Part of binding.cpp, whose helpers it uses; included there once, in
// its anonymous namespace.
using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

at::IntArrayRef lead_of(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }
std::vector<int64_t> with_last(at::IntArrayRef lead, std::initializer_list<int64_t> last) {
  auto s = lead.vec();
  s.insert(s.end(), last);
  return s;
}

uint32_t* status_word(const Tensor& t) { return reinterpret_cast<uint32_t*>(status_of(t).data_ptr()); }

struct NormArgs {
  Tensor x, res, w;
  int64_t rows, D;
  NormArgs(const char* what, const Tensor& x_, const c10::optional<Tensor>& res_, const Tensor& w_) {
    TORCH_CHECK(float_or_bf16(x_.scalar_type()) && x_.dim() >= 1 && x_.size(-1) >= 1 && x_.size(-1) <= 32768, what,
                ": x [.., D] in bf16 or fp32, D at most 32768");
    TORCH_CHECK(!res_.has_value() || (res_->sizes() == x_.sizes() && res_->scalar_type() == x_.scalar_type() && res_->device() == x_.device()), what,
                ": a residual like x");
    TORCH_CHECK(w_.dim() == 1 && w_.size(0) == x_.size(-1) && float_or_bf16(w_.scalar_type()) && w_.device() == x_.device(), what, ": weight [D] on x's device");
    x = dense(x_);
    if (res_.has_value()) res = dense(*res_);
    w = dense(w_.to(x.scalar_type()));
    D = x.size(-1);
    rows = x.numel() / D;
  }
};

std::tuple<Tensor, Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  c10::cuda::CUDAGuard g(x.device());
  const NormArgs a("add_rms_norm", x, residual, weight);
  Tensor y = at::empty_like(a.x), h = at::empty_like(a.x), rstd = at::empty(lead_of(a.x), a.x.options().dtype(at::kFloat));
  check(apb_add_rms_norm(a.x.data_ptr(), a.res.data_ptr(), a.w.data_ptr(), h.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), nullptr, nullptr, a.rows,
                         (int)a.D, (float)eps, is_bf16(a.x), stream()),
        "apb_add_rms_norm");
  count(a.rows > 0);
  return {y, h, rstd};
}
Five add_rms_norm_fp8(const Tensor& x, const c10::optional<Tensor>& residual, const Tensor& weight, double eps, bool keep) {
  c10::cuda::CUDAGuard g(x.device());
  const NormArgs a("add_rms_norm_fp8", x, residual, weight);
  const auto f32 = a.x.options().dtype(at::kFloat);
  Tensor y = keep ? at::empty_like(a.x) : at::empty({0}, a.x.options()), h = a.res.defined() ? at::empty_like(a.x) : at::empty({0}, a.x.options());
  Tensor rstd = at::empty(lead_of(a.x), f32), scale = at::empty(with_last(lead_of(a.x), {1}), f32);
  Tensor q = at::empty(a.x.sizes(), a.x.options().dtype(at::kFloat8_e4m3fn));
  check(apb_add_rms_norm(a.x.data_ptr(), a.res.defined() ? a.res.data_ptr() : nullptr, a.w.data_ptr(), a.res.defined() ? h.data_ptr() : nullptr,
                         keep ? y.data_ptr() : nullptr, rstd.data_ptr<float>(), q.data_ptr(), scale.data_ptr<float>(), a.rows, (int)a.D, (float)eps,
                         is_bf16(a.x), stream()),
        "apb_add_rms_norm");
  count(a.rows > 0);
  return {y, h, rstd, q, scale};
}
// Without ``dh`` (h is not used further on, or there is no residual) it is the plain norm's gradient: that kernel's, two operands instead of three, for the widths it
// takes (those of its forward pass) and weights of the operands' type; this one's for the others.
Two add_rms_norm_bwd(const Tensor& dy_, const c10::optional<Tensor>& dh_, const Tensor& h_, const Tensor& weight, const Tensor& rstd_) {
  c10::cuda::CUDAGuard g(h_.device());
  const NormArgs a("add_rms_norm_bwd", h_, c10::nullopt, weight);
  for (const Tensor* t : {&dy_, dh_.has_value() ? &*dh_ : &dy_})
    TORCH_CHECK(t->sizes() == h_.sizes() && t->scalar_type() == h_.scalar_type() && t->device() == h_.device(), "add_rms_norm_bwd: gradients like h");
  TORCH_CHECK(rstd_.scalar_type() == at::kFloat && rstd_.numel() == a.rows && rstd_.device() == h_.device(), "add_rms_norm_bwd: rstd fp32, one a row");
  if (!dh_.has_value() && a.rows > 0 && a.D % 8 == 0 && a.D <= 16384 && weight.scalar_type() == a.x.scalar_type())
    return op_rms_norm_bwd(dy_, h_, weight, rstd_);
  // (a weight in fp32 beside bf16 operands is taken in their type, as the plain norm takes it; its gradient is not rounded to that)
  const bool wide = weight.scalar_type() == at::kFloat;
  Tensor dx = at::empty_like(a.x), dw = at::empty({a.D}, wide ? weight.options() : a.x.options());
  if (a.rows == 0) return {dx, dw.zero_().to(weight.scalar_type())};
  Tensor dy = dense(dy_), dh = dh_.has_value() ? dense(*dh_) : Tensor(), rstd = rstd_.contiguous();
  Tensor part = at::empty({(int64_t)apb_add_rms_norm_bwd_workspace(a.rows, (int)a.D, is_bf16(a.x), num_sms())}, rstd.options());  // partial sums of dw
  check(apb_add_rms_norm_bwd(dy.data_ptr(), dh.defined() ? dh.data_ptr() : nullptr, a.x.data_ptr(), a.w.data_ptr(), rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr(),
                             part.data_ptr<float>(), a.rows, (int)a.D, is_bf16(a.x), num_sms(), stream(), status_word(a.x), wide),
        "apb_add_rms_norm_bwd");
  count(2);
  return {dx, dw.to(weight.scalar_type())};
}

Two mx8_quantize(const Tensor& x_) {
  c10::cuda::CUDAGuard g(x_.device());
  TORCH_CHECK(x_.dim() >= 1 && float_or_bf16(x_.scalar_type()), "mx8_quantize: x [.., K] in bf16 or fp32");
  Tensor x = dense(x_);
  const int64_t K = x.size(-1);
  Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar)), scales = at::empty(with_last(lead_of(x), {mx_blocks(K)}), x.options().dtype(at::kByte));
  check(apb_mx8_quantize(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), K ? x.numel() / K : 0, K, is_bf16(x), stream()), "apb_mx8_quantize");
  count(x.numel() > 0);
  return {codes, scales};
}
void mx_check(const Tensor& codes, const Tensor& scales, at::ScalarType type, const char* what) {
  TORCH_CHECK(codes.scalar_type() == type && scales.scalar_type() == at::kByte && codes.dim() >= 1 && scales.device() == codes.device() &&
                  scales.sizes() == at::IntArrayRef(with_last(lead_of(codes), {mx_blocks(codes.size(-1))})),
              what, ": ", type == at::kChar ? "int8" : type == at::kShort ? "int16" : "fp16", " codes [.., K] and uint8 scales [.., ceil(K / 32)]");
}
// What is kept of both projections: the codes' type for ``bits`` (8 or 16: whole numbers, 11: fp16 numbers), and back.
constexpr int64_t HALF_BITS = 11;
at::ScalarType code_type(int64_t bits) { return bits == 8 ? at::kChar : bits == 16 ? at::kShort : at::kHalf; }
int code_bits(at::ScalarType type) { return type == at::kChar ? 8 : type == at::kShort ? 16 : type == at::kHalf ? (int)HALF_BITS : 0; }
Tensor mx8_dequantize(const Tensor& codes_, const Tensor& scales_, at::ScalarType dtype) {
  c10::cuda::CUDAGuard g(codes_.device());
  mx_check(codes_, scales_, at::kChar, "mx8_dequantize");
  TORCH_CHECK(float_or_bf16(dtype), "mx8_dequantize: bf16 or fp32");
  Tensor codes = dense(codes_), scales = scales_.contiguous(), y = at::empty(codes.sizes(), codes.options().dtype(dtype));
  const int64_t K = codes.size(-1);
  check(apb_mx8_dequantize(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), K ? codes.numel() / K : 0, K, dtype == at::kBFloat16, stream()),
        "apb_mx8_dequantize");
  count(y.numel() > 0);
  return y;
}

// -------------------------------------------------------------------------------- the gated block
// bf16, rows of whole 16 bytes, sizes that the kernels index with 32 bits: their form; others go through the plain products in fp32.
bool gated_form(std::initializer_list<const Tensor*> ts, std::initializer_list<int64_t> widths) {
  if (native().diag_library_gemm) return false;
  for (const Tensor* t : ts)
    if (t->scalar_type() != at::kBFloat16) return false;
  for (int64_t w : widths)
    if (w == 0 || w % 8 != 0 || w > 0x1fffffff) return false;  // (twice a width is counted too)
  return true;
}
int64_t rows_of(const Tensor& t, int dims) { return c10::multiply_integers(t.sizes().slice(0, t.dim() - dims)); }
void gated_check(const Tensor& x, std::initializer_list<const Tensor*> ws, const char* what) {
  TORCH_CHECK(x.dim() >= 1 && float_or_bf16(x.scalar_type()), what, ": [.., D] in bf16 or fp32");
  for (const Tensor* w : ws)
    TORCH_CHECK(w->dim() == 2 && w->scalar_type() == x.scalar_type() && w->device() == x.device(), what, ": weights are matrices of the operand's type and device");
  for (const Tensor* w : ws) TORCH_CHECK(w->size(0) <= 0x3fffffff && w->size(1) <= 0x3fffffff, what, ": weights of at most 2^30 - 1 rows and columns");
}
// x w^T or x w in fp32
Tensor product32(const Tensor& x, const Tensor& w, bool trans) {
  const int64_t M = rows_of(x, 1), N = w.size(trans ? 0 : 1);
  if (M == 0 || N == 0 || x.size(-1) == 0) return at::zeros({M, N}, x.options().dtype(at::kFloat));
  return op_mm_nd(x.reshape({M, x.size(-1)}), w, trans, at::kFloat);
}

std::tuple<Tensor, Tensor, Tensor> gated_mm(const Tensor& x, const Tensor& w1, const Tensor& w3, int64_t act, int64_t bits) {
  c10::cuda::CUDAGuard g(x.device());
  gated_check(x, {&w1, &w3}, "gated_mm");
  const int64_t D = x.size(-1), H = w1.size(0), M = rows_of(x, 1);
  TORCH_CHECK(w1.size(1) == D && w3.sizes() == w1.sizes(), "gated_mm: x [.., D], w1 and w3 [H, D]");
  TORCH_CHECK(act >= 0 && act <= 2 && (bits == 0 || bits == 8 || bits == 16 || bits == HALF_BITS), "gated_mm: act 0 to 2, bits 0, 8 or 16, or 11 for fp16 numbers");
  const auto lead = lead_of(x);
  const auto u8 = x.options().dtype(at::kByte);
  Tensor h = at::empty(with_last(lead, {H}), x.options()), ab = at::empty({0}, x.options()), scales = at::empty({0}, u8);
  if (gated_form({&x}, {D, H}) && M > 0 && M <= 0x7fffffff) {
    if (bits) {
      ab = at::empty(with_last(lead, {2, H}), x.options().dtype(code_type(bits)));
      scales = at::empty(with_last(lead, {2, mx_blocks(H)}), u8);
    }
    Tensor x2 = as2d(x), a = as2d(w1), b = as2d(w3);
    const int err = apb_gemm_gated(x2.data_ptr(), a.data_ptr(), b.data_ptr(), h.data_ptr(), bits ? ab.data_ptr() : nullptr,
                                   bits ? scales.data_ptr() : nullptr, (int)bits, (int)M, (int)H, (int)D, x2.stride(0), a.stride(0), b.stride(0), (int)act,
                                   status_word(x), num_sms(), stream());
    if (err == 0) count();
    if (err == 0) return {h, ab, scales};
    if (err > 0) check(err, "apb_gemm_gated");
  }
  Tensor both = at::stack({product32(x, w1, true), product32(x, w3, true)}, 1);  // [M, 2, H]
  check(apb_gated_act(both.data_ptr<float>(), h.data_ptr(), M, (int)H, (int)act, is_bf16(x), stream()), "apb_gated_act");
  count(both.numel() > 0);
  if (bits == 8) {
    auto [c, s] = mx8_quantize(both);
    ab = c.view(with_last(lead, {2, H}));
    scales = s.view(with_last(lead, {2, mx_blocks(H)}));
  } else if (bits && x.scalar_type() == at::kFloat) {
    ab = both.view(with_last(lead, {2, H}));
  } else if (bits) {
    ab = at::empty(with_last(lead, {2, H}), x.options().dtype(code_type(bits)));
    scales = at::empty(with_last(lead, {2, mx_blocks(H)}), u8);
    check(apb_mx16_quantize(both.data_ptr<float>(), ab.data_ptr(), scales.data_ptr(), 2 * M, (int)H, (int)bits, stream()), "apb_mx16_quantize");
    count(both.numel() > 0);
  }
  return {h, ab, scales};
}

Two gated_dgrad(const Tensor& dy, const Tensor& w2, const Tensor& ab_, const Tensor& scales_, int64_t act) {
  c10::cuda::CUDAGuard g(dy.device());
  gated_check(dy, {&w2}, "gated_dgrad");
  const int bits = code_bits(ab_.scalar_type());  // (0: values in fp32)
  const bool codes = dy.scalar_type() == at::kBFloat16 || bits == 8;
  const int64_t N = dy.size(-1), H = w2.size(1), M = rows_of(dy, 1);
  TORCH_CHECK(w2.size(0) == N && ab_.sizes() == at::IntArrayRef(with_last(lead_of(dy), {2, H})) && ab_.device() == dy.device() &&
                  (codes ? bits != 0 : ab_.scalar_type() == at::kFloat),
              "gated_dgrad: dy [.., N], w2 [N, H], ab [.., 2, H] in 8 bits, or in 16 for bf16 and fp32 for fp32");
  if (codes) mx_check(ab_, scales_, ab_.scalar_type(), "gated_dgrad");
  TORCH_CHECK(act >= 0 && act <= 2, "gated_dgrad: act 0 to 2");
  Tensor dab = at::empty(ab_.sizes(), dy.options()), h = at::empty(with_last(lead_of(dy), {H}), dy.options());
  if (gated_form({&dy}, {N, H}) && M > 0 && M <= 0x7fffffff) {
    Tensor a = as2d(dy), b = as2d(w2), ab = dense(ab_), scales = scales_.contiguous();
    const int err = apb_gemm_gated_grad(a.data_ptr(), b.data_ptr(), ab.data_ptr(), scales.data_ptr(), bits, dab.data_ptr(), h.data_ptr(),
                                        (int)M, (int)H, (int)N, a.stride(0), b.stride(0), (int)act, status_word(dy), num_sms(), stream());
    if (err == 0) count();
    if (err == 0) return {dab, h};
    if (err > 0) check(err, "apb_gemm_gated_grad");
  }
  Tensor dh = product32(dy, w2, false), v;
  if (bits == 8) {
    v = mx8_dequantize(ab_, scales_, at::kFloat);
  } else if (codes) {
    Tensor c = ab_.contiguous(), s = scales_.contiguous();
    v = at::empty(c.sizes(), c.options().dtype(at::kFloat));
    check(apb_mx16_dequantize(c.data_ptr(), s.data_ptr(), v.data_ptr<float>(), 2 * M, (int)H, bits, stream()), "apb_mx16_dequantize");
    count(v.numel() > 0);
  } else {
    v = ab_.contiguous();
  }
  check(apb_gated_act_bwd(dh.data_ptr<float>(), v.data_ptr<float>(), dab.data_ptr(), h.data_ptr(), M, (int)H, (int)act, is_bf16(dy), stream()),
        "apb_gated_act_bwd");
  count(dh.numel() > 0);
  return {dab, h};
}

Tensor gated_dx(const Tensor& dab_, const Tensor& w1, const Tensor& w3) {
  c10::cuda::CUDAGuard g(dab_.device());
  gated_check(dab_, {&w1, &w3}, "gated_dx");
  TORCH_CHECK(dab_.dim() >= 2 && dab_.size(-2) == 2 && w1.size(0) == dab_.size(-1) && w3.sizes() == w1.sizes(), "gated_dx: dab [.., 2, H], w1 and w3 [H, D]");
  const int64_t M = rows_of(dab_, 2), H = w1.size(0), D = w1.size(1);
  const auto shape = with_last(dab_.sizes().slice(0, dab_.dim() - 2), {D});
  Tensor dab = dense(dab_);
  if (gated_form({&dab}, {D, H}) && M > 0 && M <= 0x7fffffff) {
    Tensor dx = at::empty(shape, dab.options()), a = as2d(w1), b = as2d(w3);
    const at::BFloat16* p = dab.data_ptr<at::BFloat16>();
    const int err = apb_gemm_dual(p, p + H, a.data_ptr(), b.data_ptr(), dx.data_ptr(), (int)M, (int)D, (int)H, 2 * H, a.stride(0), b.stride(0), D,
                                  status_word(dab), num_sms(), stream());
    if (err == 0) count();
    if (err == 0) return dx;
    if (err > 0) check(err, "apb_gemm_dual");
  }
  Tensor m = dab.view({M, 2, H});
  return (product32(m.select(1, 0), w1, false) + product32(m.select(1, 1), w3, false)).to(dab.scalar_type()).view(shape);
}

// One product for both: rows of da and db side by side are one operand, whose product goes to two tensors.
Two gated_wgrad(const Tensor& dab, const Tensor& x, at::ScalarType dtype) {
  c10::cuda::CUDAGuard g(dab.device());
  TORCH_CHECK(dab.dim() >= 2 && dab.size(-2) == 2 && x.dim() >= 1 && rows_of(dab, 2) == rows_of(x, 1) && float_or_bf16(x.scalar_type()) &&
                  dab.scalar_type() == x.scalar_type() && dab.device() == x.device() && float_or_bf16(dtype),
              "gated_wgrad: dab [.., 2, H] and x [.., D] of one type and as many rows");
  const int64_t M = rows_of(x, 1), H = dab.size(-1), D = x.size(-1);
  if (M == 0 || H == 0 || D == 0) return {at::zeros({H, D}, x.options().dtype(dtype)), at::zeros({H, D}, x.options().dtype(dtype))};
  if (gated_form({&dab, &x}, {H, D}) && M <= 0x7fffffff) {
    Tensor a = as2d(dab.reshape({M, 2 * H})), b = as2d(x.reshape({M, D}));
    Tensor dw1 = at::empty({H, D}, x.options().dtype(dtype)), dw3 = at::empty_like(dw1);
    const int err = apb_gemm_two(a.data_ptr(), b.data_ptr(), dw1.data_ptr(), dw3.data_ptr(), (int)H, (int)D, (int)M, a.stride(0), b.stride(0), dtype == at::kFloat,
                                 status_word(x), num_sms(), stream());
    if (err == 0) count();
    if (err == 0) return {dw1, dw3};
    if (err > 0) check(err, "apb_gemm_two");
  }
  Tensor both = dab.reshape({M, 2, H}), x2 = x.reshape({M, D});
  return {op_mm_wgrad(both.select(1, 0), x2, dtype), op_mm_wgrad(both.select(1, 1), x2, dtype)};
}

// Whether the product with w2 is the few-row kernel's, whose first loads do not wait for h, with w2 as it lies in memory (a copy would be made by the kernel
// before it): where a product of its own would be, and up to 16 rows for a round of blocks (two to an SM, of 16 columns) also where the contraction is longer; both
// products of the block, us, so / with the split kernel: 8 x 4096 x 14336 57 / 67, 16 x 4096 x 14336 70 / 73, 16 x 2048 x 14336 39 / 41; with fewer columns
// 16 x 512 x 14336 24 / 19.
bool few_rows_behind(const Tensor& h, const Tensor& w2, int64_t M, int64_t N, int64_t H) {
  return gated_form({&h}, {N, H}) && M <= 32 && apb_gemm_get_reserved_sms() == 0 &&
         (apb_gemm_rows_takes((int)M, (int)N, (int)H, num_sms()) || (M <= 16 && N >= 2048 && N <= 32 * num_sms())) &&
         w2.stride(1) == 1 && w2.stride(0) >= H && w2.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(w2.data_ptr()) % 16 == 0;
}

Five gated_ffn(const Tensor& x, const Tensor& w1, const Tensor& w3, const Tensor& w2, int64_t act, int64_t bits) {
  c10::cuda::CUDAGuard g(x.device());
  gated_check(x, {&w1, &w3, &w2}, "gated_ffn");
  TORCH_CHECK(w2.size(1) == w1.size(0), "gated_ffn: w1 and w3 [H, D], w2 [N, H]");
  auto [h, ab, scales] = gated_mm(x, w1, w3, act, bits);
  const int64_t N = w2.size(0);
  const int64_t M = rows_of(h, 1), H = h.size(-1);
  Tensor y;
  if (h.numel() == 0 || N == 0) {
    y = at::zeros(with_last(lead_of(x), {N}), x.options());
  } else if (ours(MM_ND) && few_rows_behind(h, w2, M, N, H)) {
    y = at::empty(with_last(lead_of(x), {N}), x.options());
    check(apb_gemm_rows_behind(h.data_ptr(), w2.data_ptr(), y.data_ptr(), (int)M, (int)N, (int)H, H, w2.stride(0), N, 0, num_sms(), stream()),
          "apb_gemm_rows_behind");
    count();
  } else {
    y = op_mm_nd(h, w2, true, x.scalar_type());
  }
  const auto u8 = x.options().dtype(at::kByte);
  if (bits != 8) return {y, ab, scales, at::empty({0}, u8), at::empty({0}, u8)};
  auto [xq, xs] = mx8_quantize(x);
  return {y, ab, scales, xq, xs};
}

// -------------------------------------------------------------------------------- entries
using Three = std::tuple<Tensor, Tensor, Tensor>;
Three op_add_rms_norm(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
  return ours(ADD_RMS_NORM) ? add_rms_norm(x, r, w, eps) : in_python<Three>(ADD_RMS_NORM, x, r, w, eps);
}
Two op_add_rms_norm_bwd(const Tensor& dy, const c10::optional<Tensor>& dh, const Tensor& h, const Tensor& w, const Tensor& rstd) {
  return ours(ADD_RMS_NORM_BWD) ? add_rms_norm_bwd(dy, dh, h, w, rstd) : in_python<Two>(ADD_RMS_NORM_BWD, dy, dh, h, w, rstd);
}
Five op_add_rms_norm_fp8(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w, double eps, bool keep) {
  return ours(ADD_RMS_NORM_FP8) ? add_rms_norm_fp8(x, r, w, eps, keep) : in_python<Five>(ADD_RMS_NORM_FP8, x, r, w, eps, keep);
}
Two op_mx8_quantize(const Tensor& x) { return ours(MX8_QUANTIZE) ? mx8_quantize(x) : in_python<Two>(MX8_QUANTIZE, x); }
Tensor op_mx8_dequantize(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  if (ours(MX8_DEQUANTIZE)) return mx8_dequantize(codes, scales, dtype);
  py::gil_scoped_acquire gil;
  return in_python<Tensor>(MX8_DEQUANTIZE, codes, scales, py_dtype(dtype));
}
Three op_gated_mm(const Tensor& x, const Tensor& w1, const Tensor& w3, int64_t act, int64_t bits) {
  return ours(GATED_MM) ? gated_mm(x, w1, w3, act, bits) : in_python<Three>(GATED_MM, x, w1, w3, act, bits);
}
Two op_gated_dgrad(const Tensor& dy, const Tensor& w2, const Tensor& ab, const Tensor& scales, int64_t act) {
  return ours(GATED_DGRAD) ? gated_dgrad(dy, w2, ab, scales, act) : in_python<Two>(GATED_DGRAD, dy, w2, ab, scales, act);
}
Tensor op_gated_dx(const Tensor& dab, const Tensor& w1, const Tensor& w3) {
  return ours(GATED_DX) ? gated_dx(dab, w1, w3) : in_python<Tensor>(GATED_DX, dab, w1, w3);
}
Two op_gated_wgrad(const Tensor& dab, const Tensor& x, at::ScalarType dtype) {
  if (ours(GATED_WGRAD)) return gated_wgrad(dab, x, dtype);
  py::gil_scoped_acquire gil;
  return in_python<Two>(GATED_WGRAD, dab, x, py_dtype(dtype));
}
Five op_gated_ffn(const Tensor& x, const Tensor& w1, const Tensor& w3, const Tensor& w2, int64_t act, int64_t bits) {
  return ours(GATED_FFN) ? gated_ffn(x, w1, w3, w2, act, bits) : in_python<Five>(GATED_FFN, x, w1, w3, w2, act, bits);
}
