// bf16 products with a handful of rows, sm_100a: a projection of a few tokens (decoding).
//
//   C[M, N] = X[M, K] * W[N, K]^T, M <= 32, K % 8 == 0, fp32 sums; C bf16 or fp32
//
// Bound by reading W once.  The tensor-core kernel of gemm_split.cu spends half of such a launch outside that: TMEM allocation, barriers, tiles of
// 128 rows of which a few are used, fp32 tiles added up through a cluster.  Here a block owns 16 rows of W (columns of C), its sixteen warps
// take a sixteenth of K each, and W and X go from memory to registers in the fragments of mma.sync (m16n8k16, W as the 16-row operand): a thread
// loads 8 consecutive elements of a row, which are its share of two MMAs whose k is permuted alike for both operands.  The partial sums of the
// warps meet in shared memory, in warp order: the same result every time, and shorter chains of fp32 sums than the other kernel's.
// Split kernel -> this one, us: 1 x 4096 x 4096 10.7 -> 7.3 (4.6 TB/s with the launch), 16 x 4096 x 4096 10.3 -> 8.7, 8 x 2048 x 2048 7.3 -> 3.7,
// 8 x 256 x 256 3.9 -> 1.9, 1 x 32064 x 4096 51.6 -> 42.2.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gated.cuh"
#include "launch.cuh"

namespace apb {

constexpr int ROWS_WARPS = 16, ROWS_MAX = 32, ROWS_TILE = 16;

__device__ __forceinline__ uint4 ld_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// What becomes of the sums.  ``pair``: of the 16 rows of the operand, 8 are W's and 8 a second matrix's (the two projections of a gated feed-forward block,
// N columns each).
struct RowsPlain {
  static constexpr bool PAIR = false;
  void* C;
  long long ldc;
  int out_fp32;
};
struct RowsGated {
  static constexpr bool PAIR = true;
  const __nv_bfloat16* W3;
  long long ldw3;
  __nv_bfloat16* h;
  int act;
};

// MB: blocks of 8 rows of X; U: steps of 32 elements of K whose loads are under way together; RW: warps of a block, which share K.  EARLY: the kernel before does not write W, nor can one before
// that be writing it still (it lets this one in behind its own wait), so the first loads of W do not wait for it.
template <int MB, int U, int RW, bool EARLY, typename Out>
__device__ __forceinline__ void rows_cta(const __nv_bfloat16* X, const __nv_bfloat16* W, int M, int N, int K, long long ldx, long long ldw, const Out& out) {
  constexpr int TM = 8 * MB;
  __shared__ float part[RW][TM * ROWS_TILE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 8;
  const int n0 = blockIdx.x * (Out::PAIR ? ROWS_TILE / 2 : ROWS_TILE);
  const int steps = (K + 31) / 32, s0 = steps * warp / RW, s1 = steps * (warp + 1) / RW;
  const __nv_bfloat16* w[2];
  const __nv_bfloat16* x[MB];
  bool wk[2], xk[MB];  // rows outside the matrices load nothing
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (Out::PAIR) {
      wk[i] = n0 + g < N;
      w[i] = (i ? out.W3 : W) + (wk[i] ? n0 + g : 0) * (i ? out.ldw3 : ldw) + c;
    } else {
      wk[i] = n0 + g + 8 * i < N;
      w[i] = W + (wk[i] ? n0 + g + 8 * i : 0) * ldw + c;
    }
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    xk[i] = g + 8 * i < M;
    x[i] = X + (xk[i] ? g + 8 * i : 0) * ldx + c;
  }
  float acc[MB][4] = {};
  auto load_w = [&](uint4 (&wv)[U][2], int s) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * 32;
      const bool in = s + u < s1 && k + c < K;  // (K % 8 == 0: eight elements are in or out together)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        wv[u][i] = make_uint4(0, 0, 0, 0);
        if (in && wk[i]) wv[u][i] = ld_stream(w[i] + k);
      }
    }
  };
  auto step = [&](const uint4 (&wv)[U][2], int s) {
    uint4 xv[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * 32;
      const bool in = s + u < s1 && k + c < K;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        xv[u][i] = make_uint4(0, 0, 0, 0);
        if (in && xk[i]) xv[u][i] = __ldca(reinterpret_cast<const uint4*>(x[i] + k));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 a = wv[u][0], b = wv[u][1];
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        mma_bf16(acc[m], a.x, b.x, a.y, b.y, xv[u][m].x, xv[u][m].y);
        mma_bf16(acc[m], a.z, b.z, a.w, b.w, xv[u][m].z, xv[u][m].w);
      }
    }
  };
  uint4 wv[U][2];
  int s = s0;
  if constexpr (EARLY) {
    load_w(wv, s);
    after_previous();
    step(wv, s);  // (a warp without steps has zeros)
    s += U;
  }
  for (; s < s1; s += U) {
    load_w(wv, s);
    step(wv, s);
  }
  const int m2 = (lane & 3) * 2;
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][(8 * m + m2 + (i & 1)) * ROWS_TILE + g + 8 * (i >> 1)] = acc[m][i];
  __syncthreads();
  if constexpr (Out::PAIR) {
    for (int t = threadIdx.x; t < M * (ROWS_TILE / 2); t += 32 * RW) {
      const int m = t / (ROWS_TILE / 2), n = n0 + t % (ROWS_TILE / 2), at = m * ROWS_TILE + t % (ROWS_TILE / 2);
      float a = 0.f, b = 0.f, h = 0.f;
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        a += part[i][at];
        b += part[i][at + ROWS_TILE / 2];
      }
      if (n >= N) continue;
      with_act(out.act, [&](auto act) {
        float d;
        h = act_value<decltype(act)::value>(a, d) * b;
      });
      out.h[(long long)m * N + n] = __float2bfloat16(h);
    }
  } else {
    for (int t = threadIdx.x; t < M * ROWS_TILE; t += 32 * RW) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < RW; ++i) v += part[i][t];
      const int m = t / ROWS_TILE, n = n0 + t % ROWS_TILE;
      if (n < N) {
        if (out.out_fp32) reinterpret_cast<float*>(out.C)[m * out.ldc + n] = v;
        else reinterpret_cast<__nv_bfloat16*>(out.C)[m * out.ldc + n] = __float2bfloat16(v);
      }
    }
  }
}

template <int MB, int U, int MIN_BLOCKS, bool EARLY, int RW = ROWS_WARPS>
__global__ void __launch_bounds__(32 * RW, MIN_BLOCKS)
gemm_rows_kernel(const __nv_bfloat16* X, const __nv_bfloat16* W, void* C, int M, int N, int K, long long ldx,
                 long long ldw, long long ldc, int out_fp32) {
  if (!EARLY) after_previous();
  rows_cta<MB, U, RW, EARLY>(X, W, M, N, K, ldx, ldw, RowsPlain{C, ldc, out_fp32});
}
template <int MB, int RW, int MIN_BLOCKS>
__global__ void __launch_bounds__(32 * RW, MIN_BLOCKS)
gemm_rows_gated_kernel(const __nv_bfloat16* X, const __nv_bfloat16* W, int M, int N, int K, long long ldx, long long ldw, const RowsGated out) {
  after_previous();
  rows_cta<MB, 4, RW, false>(X, W, M, N, K, ldx, ldw, out);
}

}  // namespace apb

using namespace apb;

// Whether the product is this kernel's: where it is no slower than the split kernel, both launched to overlap.  Fitted to 3478 sizes (1 to 32 rows,
// 64 <= N <= 32768, 64 <= K <= 14336): the mean loss against the better one of both is 0.2, 0.6 and 1.3 % with up to 8, 16 and 32 rows (as the line was
// drawn with launches that did not overlap: 4, 5 and 9 %, at worst a factor of four).  us in a captured graph, split / this one:
//   up to 8 rows  8 x 256 x 256 2.7 / 1.6, 8 x 4096 x 4096 10.7 / 7.4, 8 x 32064 x 4096 51 / 43.  Every round of the blocks that are resident together
//                 (two to an SM) costs as much as a launch, so that many columns need some K: 8 x 14336 x 256 5.4 / 6.3, x 1024 10.7 / 8.4.  With few
//                 columns and a long K there are too few blocks: 8 x 256 x 8192 4.9 / 6.6, 8 x 1024 x 8192 8.5 / 8.3, 1 x 512 x 8192 8.4 / 7.8.
//   up to 16      X comes from L2 once per 16 columns and is half of what a block reads: 16 x 2048 x 2048 6.1 / 4.1, 16 x 4096 x 4096 8.8 / 8.3, 16 x 512
//                 x 4096 4.2 / 5.3, 16 x 6144 x 512 5.8 / 4.8, 16 x 14336 x 512 7.2 / 8.8, x 1024 10.8 / 10.1, 16 x 4096 x 8192 15 / 16.
//   up to 32      32 x 1024 x 1024 4.1 / 3.4, 24 x 2048 x 2048 6.4 / 4.7, 32 x 4096 x 1024 6.0 / 5.8; 32 x 1024 x 2048 4.2 / 4.8, 32 x 4096 x 512 4.6 /
//                 5.3 (here it is one of the losses), 32 x 6144 x 256 4.0 / 6.4, 32 x 14336 x 256 5.5 / 11.6.
extern "C" int apb_gemm_rows_takes(int M, int N, int K, int num_sms) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 8) return 0;
  const long long round = 2ll * ROWS_TILE * num_sms;  // columns of the blocks that are resident together
  const long long size = (long long)N * K, x = (long long)M * K;
  if (M <= 8) return K <= 6144 ? N <= 2 * round || N <= 32ll * K : N >= 512 && N <= round && x <= 65536;
  if (M <= 16) return K <= 3072 ? N <= (K >= 192 ? 2 : 1) * round || N <= 20ll * K : K <= 6144 && N >= 1024 && N <= round;
  return M <= ROWS_MAX && (size <= 8192 || (K >= 192 && x <= 49152 && size <= 2048 * 2048 && N <= 8ll * K));
}

namespace apb {
template <bool EARLY>
static int gemm_rows(const void* X, const void* W, void* C, int M, int N, int K, long long ldx, long long ldw, long long ldc, int out_fp32, int num_sms,
                     cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (M > ROWS_MAX || K <= 0 || (K & 7) || (ldx & 7) || (ldw & 7) || ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(W)) & 15)) return 3;
  const unsigned grid = (unsigned)((N + ROWS_TILE - 1) / ROWS_TILE);
  auto launch = [&](auto kern, int warps = ROWS_WARPS) {
    launch_after(kern, grid, 32 * warps, 0, st, (const __nv_bfloat16*)X, (const __nv_bfloat16*)W, C, M, N, K, ldx, ldw, ldc, out_fp32);
  };
  // Two blocks to an SM and three steps under way; where there is no second block and K is long enough for it, four (8 x 2048 x 2048 4.0 -> 3.7 us, 32
  // x 2048 x 2048 6.4 -> 5.3; 8 x 512 x 512 2.0 -> 2.2).  EARLY: four whatever K is, as they are on their way while the kernel before ends (both
  // products of a gated block with up to 2368 columns of this one, 308 sizes, 6 % less in the mean); more than 16 rows in two blocks of eight warps, which do
  // not spill (7 % less).
  const bool deep = grid <= (unsigned)num_sms && (EARLY || K >= 2048);
  if (M <= 8) {
    deep ? launch(gemm_rows_kernel<1, 4, 1, EARLY>) : launch(gemm_rows_kernel<1, 3, 2, EARLY>);
  } else if constexpr (EARLY) {
    if (M <= 16) deep ? launch(gemm_rows_kernel<2, 4, 1, true>) : launch(gemm_rows_kernel<2, 3, 2, true>);
    else deep ? launch(gemm_rows_kernel<4, 4, 1, true>) : launch(gemm_rows_kernel<4, 4, 2, true, 8>, 8);
  } else {
    if (M <= 16) launch(gemm_rows_kernel<2, 3, 2, false>);
    else deep ? launch(gemm_rows_kernel<4, 4, 1, false>) : launch(gemm_rows_kernel<4, 3, 2, false>);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
}  // namespace apb

// X, W: 16-byte bases and rows.  Returns 0, or an argument / launch error (nothing launched).
extern "C" int apb_gemm_rows(const void* X, const void* W, void* C, int M, int N, int K, long long ldx, long long ldw, long long ldc, int out_fp32,
                             int num_sms, cudaStream_t st) {
  return gemm_rows<false>(X, W, C, M, N, K, ldx, ldw, ldc, out_fp32, num_sms, st);
}
// The same behind a kernel of ``launch_after`` that has made X and does not write W, whatever that one is: the first loads of W do not wait for its end.
extern "C" int apb_gemm_rows_behind(const void* X, const void* W, void* C, int M, int N, int K, long long ldx, long long ldw, long long ldc, int out_fp32,
                                    int num_sms, cudaStream_t st) {
  return gemm_rows<true>(X, W, C, M, N, K, ldx, ldw, ldc, out_fp32, num_sms, st);
}

// h[M, H] = act(X W1^T) * (X W3^T) (gated.cuh).
extern "C" int apb_gemm_rows_gated(const void* X, const void* W1, const void* W3, void* h, int M, int H, int K, long long ldx, long long ldw1,
                                   long long ldw3, int act, int num_sms, cudaStream_t st) {
  if (M <= 0 || H <= 0) return 0;
  if (M > ROWS_MAX || K <= 0 || (K & 7) || ((ldx | ldw1 | ldw3) & 7) ||
      ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(W1) | reinterpret_cast<uintptr_t>(W3)) & 15))
    return 3;
  const unsigned grid = (unsigned)((H + ROWS_TILE / 2 - 1) / (ROWS_TILE / 2));
  const RowsGated out{(const __nv_bfloat16*)W3, ldw3, (__nv_bfloat16*)h, act};
  auto launch = [&](auto kern, int warps) {
    launch_after(kern, grid, 32 * warps, 0, st, (const __nv_bfloat16*)X, (const __nv_bfloat16*)W1, M, H, K, ldx, ldw1, out);
  };
  // Blocks of eight warps with four steps under way, two or three to an SM (three have 80 registers a thread, which pays with more than eight rows only where
  // there are as many blocks); sixteen warps where an SM has one block.  Against the plain product's blocks (sixteen warps, three steps, two to an SM), us: 1 x
  // 4096 x 14336 42.7 -> 37.0, 8 x 4096 x 14336 44.2 -> 38.0, 1 x 2048 x 8192 16.0 -> 12.4, 8 x 1024 x 4096 6.4 -> 4.9, 16 x 1024 x 2816 6.5 -> 4.4, 32 x 512 x
  // 2048 5.7 -> 3.9: a block of half the length waits half as long for its own end.  In 385 sizes 2 to 4 % from the best of six such forms.
  const bool two = grid <= 2u * num_sms;
  if (M <= 8) grid <= (unsigned)num_sms ? launch(gemm_rows_gated_kernel<1, 16, 1>, 16) : launch(gemm_rows_gated_kernel<1, 8, 2>, 8);
  else if (M <= 16) two ? launch(gemm_rows_gated_kernel<2, 8, 2>, 8) : launch(gemm_rows_gated_kernel<2, 8, 3>, 8);
  else two ? launch(gemm_rows_gated_kernel<4, 8, 2>, 8) : launch(gemm_rows_gated_kernel<4, 8, 3>, 8);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
