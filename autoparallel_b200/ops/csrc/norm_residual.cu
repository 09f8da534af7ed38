// The residual's addition with the norm after it, sm_100a.
//
//   forward    h = round(x + residual)    r = 1 / sqrt(mean(h^2) + eps)    y = h r w
//              in 8 bits: q = e4m3(y / s), s = max |y| of the row / 448 (1 where that maximum is below 2^-100)
//   backward   with n = h r and g = dy w:  dx = dresidual = dh + r (g - n mean(g n))    dw = sum over rows of dy n
//
// Both are bound by memory: x and residual are read once, h and y (or q) written once; backward h, dy and dh are read and dx is written.  A row stays in
// registers from its load to the last result.  The sum of squares is that of the plain norm's kernel (elementwise.cu), thread by thread, so that y has the bits
// of rms_norm(h).
#include <cuda_fp8.h>

#include "rowwise.cuh"

namespace apb {

typedef __nv_bfloat16 bf16;

// N elements of a row from column ``c`` on: a vector, or (N = 1, widths that 8 does not divide) one.
template <typename T, int N> struct Piece;
template <typename T> struct Piece<T, 8> : Vec8<T> {};
template <typename T> struct Piece<T, 1> {
  T v;
  __device__ void load(const T* p) { v = *p; }
  __device__ void store(T* p) const { *p = v; }
  __device__ void to_float(float (&f)[1]) const { f[0] = float(v); }
  __device__ void from_float(const float (&f)[1]) { v = T(f[0]); }
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {  // (satfinite: what rounding puts a hair above 448 is 448)
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
template <int N>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[N]) {
  if constexpr (N == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(e4m3x2(f[0], f[1]) | e4m3x2(f[2], f[3]) << 16, e4m3x2(f[4], f[5]) | e4m3x2(f[6], f[7]) << 16);
  } else {
    *p = (uint8_t)(e4m3x2(f[0], 0.f) & 255u);
  }
}

struct AddNormOut {
  void *h, *y;  // h: null where there is no residual; y: null where only q is wanted
  float* rstd;
  uint8_t* q;  // null: no 8-bit result
  float* scale;
};

// largest of the block's values (bits of magnitudes: a NaN is larger than everything); ``red``: 32 words
__device__ __forceinline__ uint32_t block_top(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, l < nw ? red[l] : 0u);
}

// A warp (WARP_ROWS) or a block has a row, each thread up to NP pieces of N elements.
template <typename T, int N, int NP, bool WARP_ROWS, bool FP8>
__global__ void __launch_bounds__(WARP_ROWS ? 256 : 1024) add_rms_norm_kernel(const T* x, const T* res, const T* w, const AddNormOut o, long long rows, int D,
                                                                              float eps) {
  after_previous();
  __shared__ float red[32];
  __shared__ uint32_t red_top[32];
  const int tpr = WARP_ROWS ? 32 : blockDim.x;
  const int t = WARP_ROWS ? (threadIdx.x & 31) : threadIdx.x;
  const long long step = WARP_ROWS ? gridDim.x * (long long)(blockDim.x >> 5) : gridDim.x;
  for (long long row = WARP_ROWS ? blockIdx.x * (long long)(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; row < rows; row += step) {
    const T* xr = x + row * D;
    const T* rr = res + row * D;
    Piece<T, N> v[NP], u[NP];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (t + j * tpr) * N;
      if (c < D) {
        v[j].load(xr + c);
        if (res != nullptr) u[j].load(rr + c);
      }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (t + j * tpr) * N;
      if (c < D) {
        float f[N];
        v[j].to_float(f);
        if (res != nullptr) {
          float g[N];
          u[j].to_float(g);
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] += g[i];
          v[j].from_float(f);  // h as it is stored is what the norm is taken of
          v[j].store(reinterpret_cast<T*>(o.h) + row * D + c);
          v[j].to_float(f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) ss += f[i] * f[i];
      }
    }
    ss = WARP_ROWS ? warp_sum(ss) : block_sum(ss, red);
    const float r = rsqrtf(ss / D + eps);
    if (t == 0) o.rstd[row] = r;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (t + j * tpr) * N;
      if (c < D) {
        Piece<T, N> wv;
        wv.load(w + c);
        float f[N], g[N];
        v[j].to_float(f);
        wv.to_float(g);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = f[i] * r * g[i];
        if (FP8) {
#pragma unroll
          for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
        }
        if (!FP8 || o.y != nullptr) {
          Piece<T, N> ov;
          ov.from_float(f);
          ov.store(reinterpret_cast<T*>(o.y) + row * D + c);
        }
      }
    }
    if (FP8) {
      const float amax = __uint_as_float(WARP_ROWS ? __reduce_max_sync(0xffffffffu, top) : block_top(top, red_top));
      const float s = amax < 0x1p-100f ? 1.f : __fdiv_rn(amax, 448.f);
      const float inv = __frcp_rn(s);
      if (t == 0) o.scale[row] = s;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int c = (t + j * tpr) * N;
        if (c < D) {
          Piece<T, N> wv;
          wv.load(w + c);
          float f[N], g[N];
          v[j].to_float(f);
          wv.to_float(g);
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] = f[i] * r * g[i] * inv;
          store_e4m3<N>(o.q + row * D + c, f);
        }
      }
    }
  }
}

// Backward.  Blocks take rows in turn and keep their sums of dw in registers; each leaves one row of partial sums, which rms_dw_kernel adds up in order: the
// same result every time.
template <typename T, int N, int NP>
__global__ void __launch_bounds__(1024) add_rms_norm_bwd_kernel(const T* dy, const T* dh, const T* h, const T* w, const float* rstd, T* dx, float* part,
                                                                long long rows, int D) {
  after_previous();
  __shared__ float red[32];
  float dw[NP][N], wf[NP][N];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) dw[j][i] = wf[j][i] = 0.f;
    if (c < D) {
      Piece<T, N> wv;
      wv.load(w + c);
      wv.to_float(wf[j]);
    }
  }
  const float inv_d = 1.f / D;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    Piece<T, N> hv[NP], gv[NP], ev[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (threadIdx.x + j * blockDim.x) * N;
      if (c < D) {
        hv[j].load(h + row * D + c);
        gv[j].load(dy + row * D + c);
        ev[j].load(dh + row * D + c);
      }
    }
    const float r = rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (threadIdx.x + j * blockDim.x) * N;
      if (c < D) {
        float hf[N], gf[N];
        hv[j].to_float(hf);
        gv[j].to_float(gf);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float gh = gf[i] * hf[i];
          dw[j][i] = fmaf(gh, r, dw[j][i]);
          dot = fmaf(gh, wf[j][i], dot);
        }
      }
    }
    dot = block_sum(dot, red);
    const float k = r * r * r * dot * inv_d;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = (threadIdx.x + j * blockDim.x) * N;
      if (c < D) {
        float hf[N], gf[N], ef[N];
        hv[j].to_float(hf);
        gv[j].to_float(gf);
        ev[j].to_float(ef);
#pragma unroll
        for (int i = 0; i < N; ++i) ef[i] += fmaf(gf[i], r * wf[j][i], -hf[i] * k);
        ev[j].from_float(ef);
        ev[j].store(dx + row * D + c);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int c = (threadIdx.x + j * blockDim.x) * N;
    if (c < D) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[(long long)blockIdx.x * D + c + i] = dw[j][i];
    }
  }
}

constexpr int ADD_NORM_MAX = 32768;  // columns: 1024 threads with 32 elements each

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

struct BwdPlan {
  int n, threads, np, grid;
};
// Threads of a row: two vectors each (or 8 single elements) up to 1024 threads.  Blocks: as many as an SM holds with a few rows in flight, at least four rows
// to each where there are enough, so that few rows do not leave as many partial rows of dw.
static BwdPlan bwd_plan(long long rows, int D, int num_sms) {
  BwdPlan p;
  p.n = D % 8 == 0 ? 8 : 1;
  const int pieces = (D + p.n - 1) / p.n, per = p.n == 8 ? 2 : 8;
  p.threads = 32;
  while (p.threads * per < pieces && p.threads < 1024) p.threads *= 2;
  const int np = (pieces + p.threads - 1) / p.threads;
  p.np = p.n == 8 ? (np <= 1 ? 1 : np <= 2 ? 2 : 4) : (np <= 8 ? 8 : 32);
  const int per_sm = p.threads >= 1024 ? 1 : 1024 / p.threads > 16 ? 16 : 1024 / p.threads;
  const long long cap = (long long)num_sms * per_sm, quarter = (rows + 3) / 4, least = rows < num_sms ? rows : num_sms;
  long long g = quarter < cap ? quarter : cap;
  if (g < least) g = least;
  p.grid = (int)g;
  return p;
}

template <typename T>
static cudaError_t launch_fwd(const void* x, const void* res, const void* w, const AddNormOut& o, long long rows, int D, float eps, int num_sms,
                              cudaStream_t st) {
  const bool vec = D % 8 == 0, fp8 = o.q != nullptr;
  auto launch = [&](auto kern, unsigned grid, int threads) {
    return launch_after(kern, grid, threads, 0, st, (const T*)x, (const T*)res, (const T*)w, o, rows, D, eps);
  };
#define APB_ADD_NORM(N, NP, WARP, GRID, THREADS)                                                         \
  return fp8 ? launch(add_rms_norm_kernel<T, N, NP, WARP, true>, GRID, THREADS) : launch(add_rms_norm_kernel<T, N, NP, WARP, false>, GRID, THREADS)
  if (vec && D <= 1024) {  // a warp to a row, eight rows a block
    const unsigned grid = (unsigned)((rows + 7) / 8);
    const int np = (D + 255) / 256;
    if (np == 1) APB_ADD_NORM(8, 1, true, grid, 256);
    if (np == 2) APB_ADD_NORM(8, 2, true, grid, 256);
    APB_ADD_NORM(8, 4, true, grid, 256);
  }
  if (vec) {
    int threads = 256;
    while (threads * 8 * 4 < D && threads < 1024) threads *= 2;
    const int np = (D + threads * 8 - 1) / (threads * 8);
    const unsigned grid = (unsigned)rows;
    if (np == 1) APB_ADD_NORM(8, 1, false, grid, threads);
    if (np == 2) APB_ADD_NORM(8, 2, false, grid, threads);
    APB_ADD_NORM(8, 4, false, grid, threads);
  }
  int threads = 32;
  while (threads * 8 < D && threads < 1024) threads *= 2;
  const unsigned grid = (unsigned)rows;
  if (D <= threads * 8) APB_ADD_NORM(1, 8, false, grid, threads);
  APB_ADD_NORM(1, 32, false, grid, threads);
#undef APB_ADD_NORM
}

template <typename T>
static cudaError_t launch_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx, void* dw, float* part,
                              long long rows, int D, int num_sms, cudaStream_t st) {
  const BwdPlan p = bwd_plan(rows, D, num_sms);
  auto launch = [&](auto kern) {
    return launch_after(kern, p.grid, p.threads, 0, st, (const T*)dy, (const T*)dh, (const T*)h, (const T*)w, rstd, (T*)dx, part, rows, D);
  };
  cudaError_t e;
  if (p.n == 8) e = p.np == 1 ? launch(add_rms_norm_bwd_kernel<T, 8, 1>) : p.np == 2 ? launch(add_rms_norm_bwd_kernel<T, 8, 2>) : launch(add_rms_norm_bwd_kernel<T, 8, 4>);
  else e = p.np == 8 ? launch(add_rms_norm_bwd_kernel<T, 1, 8>) : launch(add_rms_norm_bwd_kernel<T, 1, 32>);
  if (e != cudaSuccess) return e;
  return launch_after(rms_dw_kernel<T>, (unsigned)((D + 31) / 32), 1024, 0, st, (const float*)part, (T*)dw, p.grid, D);
}

}  // namespace apb

using namespace apb;

// Widths that 8 divides take vectors and need 16-byte bases.  Returns 0, or an argument / launch error (nothing launched).
extern "C" int apb_add_rms_norm(const void* x, const void* res, const void* w, void* h, void* y, float* rstd, void* q, float* scale, long long rows, int D,
                                float eps, int is_bf16, int num_sms, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (D <= 0 || D > ADD_NORM_MAX || rows > 0x7fffffffll || (res != nullptr && h == nullptr) || (y == nullptr && q == nullptr)) return 3;
  for (const void* p : {x, res, w, (const void*)h, (const void*)y, (const void*)q})
    if (off16(p)) return 3;
  const AddNormOut o{h, y, rstd, (uint8_t*)q, scale};
  const cudaError_t e = is_bf16 ? launch_fwd<bf16>(x, res, w, o, rows, D, eps, num_sms, st) : launch_fwd<float>(x, res, w, o, rows, D, eps, num_sms, st);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4;
}

// floats of workspace: a partial row of dw per block
extern "C" long long apb_add_rms_norm_bwd_workspace(long long rows, int D, int num_sms) {
  return rows <= 0 || D <= 0 ? 0 : (long long)bwd_plan(rows, D, num_sms).grid * D;
}
extern "C" int apb_add_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx, void* dw, float* part,
                                    long long rows, int D, int is_bf16, int num_sms, cudaStream_t st) {
  if (rows <= 0 || D <= 0 || D > ADD_NORM_MAX) return 3;
  for (const void* p : {dy, dh, h, w, (const void*)dx})
    if (off16(p)) return 3;
  const cudaError_t e = is_bf16 ? launch_bwd<bf16>(dy, dh, h, w, rstd, dx, dw, part, rows, D, num_sms, st)
                                : launch_bwd<float>(dy, dh, h, w, rstd, dx, dw, part, rows, D, num_sms, st);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4;
}
