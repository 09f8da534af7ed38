// The products of a gated feed-forward block, sm_100a:
//
//   apb_gemm_gated        h = act(x w1^T) * (x w3^T), and codes of x w1^T and x w3^T                               x [M, K], w [H, K]
//   apb_gemm_gated_grad   from dh = dy w2: da, db and h again (gated.cuh)                                            dy [M, K], w2 [K, H]
//   apb_gemm_dual         dx = da w1 + db w3                                                                         da, db [M, K], w [K, N]
//   apb_gemm_two          dw1 = da^T x, dw3 = db^T x, da and db side by side in one operand                          dab [K, 2 H], x [K, N]
//
// They are the bodies of the plain products (gemm_core.cuh, gemm_split.cuh) with other ends, so tiles, CTA pairs, slices and their choice are the same: a tile of
// both projections counts as one of a product with 2 H columns, the two contractions of dx as one of twice the length.  The two gradients are one product with 2 H rows whose
// halves go to two tensors.
#include "gemm_split.cuh"

extern "C" {
int apb_gemm_resident_pairs(int num_sms);
int apb_gemm_get_reserved_sms();
int apb_gemm_get_dynamic_tiles();
int apb_gemm_get_pair_stages();
int apb_gemm_get_pair_mode();
void apb_gemm_split_choice(int G, int M, int N, int K, int num_sms, int reserved, int* bn, int* s);
int apb_gemm_rows_takes(int M, int N, int K, int num_sms);
int apb_gemm_rows_gated(const void* X, const void* W1, const void* W3, void* h, int M, int H, int K, long long ldx, long long ldw1, long long ldw3,
                        int act, int num_sms, cudaStream_t st);
}

namespace apb {

// A_MN, B_MN: as stored; WIDE: gemm_core.cuh
template <bool A_MN, bool B_MN, bool WIDE, typename Ext>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GEMM_PLAIN_THREADS, 1)
gemm_ext_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p, const __grid_constant__ Ext ext) {
  extern __shared__ uint8_t smem_raw[];
  FuseParams f{};
  gemm_cta<A_MN, B_MN, FUSE_NONE, true, false, 0, false, WIDE>(tmA, tmB, p, f, blockIdx.x, gridDim.x, smem_raw, ext);
}
template <bool A_MN, bool B_MN, typename Ext>
__global__ void __launch_bounds__(GEMM_PLAIN_THREADS, 1)
gemm_ext_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p, const __grid_constant__ Ext ext) {
  extern __shared__ uint8_t smem_raw[];
  FuseParams f{};
  gemm_cta<A_MN, B_MN, FUSE_NONE>(tmA, tmB, p, f, blockIdx.x, gridDim.x, smem_raw, ext);
}
template <bool A_MN, bool B_MN, int BN_T, typename Ext>
__global__ void __launch_bounds__(SPLIT_THREADS, 1)
gemm_ext_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p,
                      const __grid_constant__ Ext ext) {
  split::gemm_cta<A_MN, B_MN, BN_T, false>(tmA, tmB, p, ext);
}

struct Operand {  // a 16-bit matrix; ``inner`` contiguous
  const void* ptr;
  long long inner, outer, ld;
  int map(CUtensorMap* m, int box) const { return make_map(m, ptr, (uint64_t)inner, (uint64_t)outer, (uint64_t)ld, (uint32_t)box); }
};

// One product with 128 rows of A, ``b_box`` rows (of a K-major B) or columns a tile.  ``second``: maps of the second operands, given the tile.
template <bool A_MN, bool B_MN, typename Ext, typename Second>
int launch_ext(const Operand& A, const Operand& B, GemmParams p, Ext ext, int num_sms, cudaStream_t stream, Second second) {
  constexpr bool HALVES = Ext::KIND == EXT_GATED;  // half of a tile's rows of B are the second matrix's
  if (((reinterpret_cast<uintptr_t>(A.ptr) | reinterpret_cast<uintptr_t>(B.ptr)) & 15) || ((A.ld | B.ld) & 7)) return 3;
  const int reserved = apb_gemm_get_reserved_sms();
  CUtensorMap tmA, tmB;
  int e = A.map(&tmA, A_MN ? BK : BM);
  if (e) return e;
  auto maps = [&](int b_box) {
    const int e2 = B.map(&tmB, b_box);
    return e2 ? e2 : second(ext, b_box);
  };
  int bn = 0, s = 0;
  if (apb_gemm_get_pair_mode()) apb_gemm_split_choice(0, p.M, p.N, p.K, num_sms, reserved, &bn, &s);
  p.num_m_tiles = (p.M + BM - 1) / BM;
  if (bn) {
    e = maps(B_MN ? BK : HALVES ? bn / 2 : bn);
    if (e) return e;
    p.num_n_tiles = (p.N + bn - 1) / bn;
    auto launch = [&](auto kern) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SPLIT_SMEM_BYTES) != cudaSuccess) return 4;
      cudaLaunchAttribute attrs[2];
      attrs[0].id = cudaLaunchAttributeClusterDimension;
      attrs[0].val.clusterDim.x = (unsigned)s;
      attrs[0].val.clusterDim.y = 1;
      attrs[0].val.clusterDim.z = 1;
      attrs[1] = overlap_attribute();
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(p.num_m_tiles * p.num_n_tiles * s));
      cfg.blockDim = dim3(SPLIT_THREADS);
      cfg.dynamicSmemBytes = SPLIT_SMEM_BYTES;
      cfg.stream = stream;
      cfg.attrs = attrs;
      cfg.numAttrs = apb_gemm_makes_room() ? 1 : 2;
      return cudaLaunchKernelEx(&cfg, kern, tmA, tmB, p, ext) == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4;
    };
    return bn == 64 ? launch(gemm_ext_split_kernel<A_MN, B_MN, 64, Ext>) : bn == 128 ? launch(gemm_ext_split_kernel<A_MN, B_MN, 128, Ext>)
                                                                              : launch(gemm_ext_split_kernel<A_MN, B_MN, 256, Ext>);
  }
  p.num_n_tiles = (p.N + BN - 1) / BN;
  const bool pair = apb_gemm_get_pair_mode() && pair_shape(p.M, p.N, p.K);
  e = maps(B_MN ? BK : pair || HALVES ? BN / 2 : BN);
  if (e) return e;
  auto launch = [&](auto kern, int grid) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_PLAIN_SMEM_BYTES) != cudaSuccess) return 4;
    return launch_after(kern, grid, GEMM_PLAIN_THREADS, GEMM_PLAIN_SMEM_BYTES, stream, tmA, tmB, p, ext) == cudaSuccess &&
                   cudaGetLastError() == cudaSuccess
               ? 0
               : 4;
  };
  if (pair) {
    int resident = apb_gemm_resident_pairs(num_sms) - reserved / 2;
    if (resident < 1) resident = 1;
    const bool wide = set_pair_tiles(p, (p.M + 2 * BM - 1) / (2 * BM), resident, true);
    const int units = 2 * p.all_tiles - p.whole_tiles, grid = 2 * (units < resident ? units : resident);
    return wide ? launch(gemm_ext_pair_kernel<A_MN, B_MN, true, Ext>, grid) : launch(gemm_ext_pair_kernel<A_MN, B_MN, false, Ext>, grid);
  }
  set_tile_order(p, p.num_m_tiles, p.num_n_tiles);
  const int tiles = p.num_m_tiles * p.num_n_tiles, usable = num_sms - reserved > 0 ? num_sms - reserved : 1;
  return launch(gemm_ext_kernel<A_MN, B_MN, Ext>, tiles < usable ? tiles : usable);
}

static GemmParams ext_params(int M, int N, int K, uint32_t* status) {
  GemmParams p{};
  p.M = M; p.N = N; p.K = K;
  p.status = status;
  return p;
}

// Shapes of these kernels: rows of whole 16 bytes.  Where GEMMs are set to hand out their tiles at run time or to leave shared memory free for
// communication kernels, plain products do that (-1: the caller's).
static int ext_takes(int M, int H, int K, bool a_mn = false) {
  if (M <= 0 || H <= 0 || K <= 0 || (H & 7) || ((a_mn ? M : K) & 7)) return 3;
  return apb_gemm_get_dynamic_tiles() || apb_gemm_get_pair_stages() != PAIR_STAGES ? -1 : 0;
}
static bool off16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return true;
  return false;
}

}  // namespace apb

using namespace apb;

// Whether a call is the few-row kernel's: as a plain product with 2 H columns, and with up to 8 rows and many columns also where the contraction is long.  385 sizes
// (1 to 32 rows, 256 <= K <= 4096, 256 <= H <= 28672): 1 to 3 % from the better one of both; few-row / split kernel, us: 1 x 4096 x 14336 37 / 42, 8 x 4096 x 5632
// 17 / 19, 1 x 8192 x 28672 144 / 195, 12 x 2048 x 5632 12 / 14, 32 x 1024 x 1024 3.7 / 5.0; 16 x 4096 x 14336 46 / 42, 32 x 2048 x 14336 36 / 24.
static bool few_rows(int M, int H, int K, int num_sms) {
  return M <= 32 && (apb_gemm_rows_takes(M, 2 * H, K, num_sms) || (M <= 8 && H >= 4096));
}

// ``bits`` 0, or 8, 16 or MX_HALF: the codes ``ab`` [M, 2, H] and ``scales`` [M, 2, ceil(H / 32)] are kept.  Returns 0, -1 (the caller's plain products), > 0: argument or
// driver error (nothing launched).
extern "C" int apb_gemm_gated(const void* x, const void* w1, const void* w3, void* h, void* ab, void* scales, int bits, int M, int H, int K,
                              long long ldx, long long ldw1, long long ldw3, int act, uint32_t* status, int num_sms, cudaStream_t stream) {
  const int no = ext_takes(M, H, K);
  if (no) return no;
  if (off16({x, w1, w3, h, ab}) || ((ldx | ldw1 | ldw3) & 7)) return 3;
  if (H > 0x3fffffff || (bits != 0 && bits != 8 && bits != 16 && bits != MX_HALF) || (bits != 0 && (ab == nullptr || scales == nullptr))) return 3;
  if (bits == 0 && apb_gemm_get_reserved_sms() == 0 && few_rows(M, H, K, num_sms))
    return apb_gemm_rows_gated(x, w1, w3, h, M, H, K, ldx, ldw1, ldw3, act, num_sms, stream);
  auto launch = [&](auto ext) {
    ext.out = GatedOut{(__nv_bfloat16*)h, ab, (uint8_t*)scales, act};
    return launch_ext<false, false>(Operand{x, K, M, ldx}, Operand{w1, K, H, ldw1}, ext_params(M, 2 * H, K, status), ext, num_sms, stream,
                             [&](auto& e, int box) { return Operand{w3, K, H, ldw3}.map(&e.tmB2, box); });
  };
  return bits == 0 ? launch(GatedExt<0>{}) : bits == 8 ? launch(GatedExt<8>{}) : bits == 16 ? launch(GatedExt<16>{}) : launch(GatedExt<MX_HALF>{});
}

extern "C" int apb_gemm_gated_grad(const void* dy, const void* w2, const void* ab, const void* scales, int bits, void* dab, void* h, int M, int H,
                                   int K, long long ldy, long long ldw, int act, uint32_t* status, int num_sms, cudaStream_t stream) {
  const int no = ext_takes(M, H, K);
  if (no) return no;
  if (off16({dy, w2, ab, dab, h}) || (bits != 8 && bits != 16 && bits != MX_HALF) || ab == nullptr || scales == nullptr) return 3;
  const GatedGrad g{ab, (const uint8_t*)scales, (__nv_bfloat16*)dab, (__nv_bfloat16*)h, act};
  const Operand A{dy, K, M, ldy}, B{w2, H, K, ldw};
  const GemmParams p = ext_params(M, H, K, status);
  auto none = [](auto&, int) { return 0; };
  return bits == 8    ? launch_ext<false, true>(A, B, p, GradExt<8>{g}, num_sms, stream, none)
         : bits == 16 ? launch_ext<false, true>(A, B, p, GradExt<16>{g}, num_sms, stream, none)
                      : launch_ext<false, true>(A, B, p, GradExt<MX_HALF>{g}, num_sms, stream, none);
}

// C[M, N] = a1[M, K] b1[K, N] + a2[M, K] b2[K, N], bf16; one accumulation over both contractions.
extern "C" int apb_gemm_dual(const void* a1, const void* a2, const void* b1, const void* b2, void* C, int M, int N, int K, long long lda, long long ldb1,
                             long long ldb2, long long ldc, uint32_t* status, int num_sms, cudaStream_t stream) {
  const int no = ext_takes(M, N, K);
  if (no) return no;
  if (off16({a1, a2, b1, b2, C}) || ((ldb1 | ldb2 | ldc) & 7)) return 3;
  const int both = 2 * ((K + BK - 1) / BK) * BK;
  GemmParams p = ext_params(M, N, both, status);
  p.C = C;
  p.ldc = ldc;
  p.vec_store = 1;
  return launch_ext<false, true>(Operand{a1, K, M, lda}, Operand{b1, N, K, ldb1}, p, DualExt{}, num_sms, stream, [&](DualExt& e, int box) {
    const int bad = Operand{a2, K, M, lda}.map(&e.tmA2, BM);
    return bad ? bad : Operand{b2, N, K, ldb2}.map(&e.tmB2, box);
  });
}

// c1[H, N] = a1^T b, c2[H, N] = a2^T b, bf16 or fp32: ``A`` [K, 2 H] has a1 and a2 side by side, ``B`` [K, N].
extern "C" int apb_gemm_two(const void* A, const void* B, void* c1, void* c2, int H, int N, int K, long long lda, long long ldb, int out_fp32,
                            uint32_t* status, int num_sms, cudaStream_t stream) {
  if (H > 0x3fffffff) return 3;
  const int no = ext_takes(H, N, K, true);
  if (no) return no;
  if (off16({A, B, c1, c2})) return 3;
  GemmParams p = ext_params(2 * H, N, K, status);
  p.C = c1;
  p.ldc = N;
  p.out_fp32 = out_fp32;
  p.vec_store = 1;
  const long long behind = (long long)H * N * (out_fp32 ? 4 : 2);
  const TwoExt ext{H, (long long)(reinterpret_cast<intptr_t>(c2) - reinterpret_cast<intptr_t>(c1)) - behind};
  return launch_ext<true, true>(Operand{A, 2 * H, K, lda}, Operand{B, N, K, ldb}, p, ext, num_sms, stream, [](auto&, int) { return 0; });
}
