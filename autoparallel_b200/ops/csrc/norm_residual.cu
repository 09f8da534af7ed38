// The residual's addition with the norm after it, sm_100a.
//
//   forward    h = round(x + residual)    r = 1 / sqrt(mean(h^2) + eps)    y = h r w
//              in 8 bits: q = e4m3(y / s), s = max |y| of the row / 448 (1 where that maximum is below 2^-100)
//   backward   with n = h r and g = dy w:  dx = dresidual = dh + r (g - n mean(g n))    dw = sum over rows of dy n    (dh: null where h is not used)
//
// Both are bound by memory: x and residual are read once, h and y (or q) written once; backward h, dy and dh are read and dx is written.  A row stays in
// registers from its load to the last result.  The sum of squares is that of the plain norm's kernel (elementwise.cu), thread by thread, so that y has the bits
// of rms_norm(h).
#include <cuda_fp8.h>

#include <type_traits>

#include "ptx.cuh"
#include "rowwise.cuh"

namespace apb {

typedef __nv_bfloat16 bf16;

// Eight elements of a row at a time.  Rows of widths that 8 does not divide (EVEN = false) begin anywhere, but all tensors of a call in the same way, so the
// vectors are those of the whole tensor: a row's first one begins ``lead`` elements before it.  What a vector has of the neighbouring rows is read as zeros
// and not written; only the weight's vectors lie off the boundaries, and its elements are read one by one.
template <typename T, bool EVEN>
struct Row {
  long long base, total;  // first element of the row, elements of the tensor
  int D, lead;
  __device__ __forceinline__ Row(long long row, long long rows, int D_) : base(row * D_), total(rows * D_), D(D_), lead(EVEN ? 0 : (int)(base & 7)) {}
  __device__ __forceinline__ int col(int vec) const { return vec * 8 - lead; }  // of its first element; below 0: some are the row's before
  __device__ __forceinline__ bool whole(int c) const { return EVEN || (c >= 0 && c + 8 <= D); }
  __device__ __forceinline__ void load(Vec8<T>& v, const T* p, int c) const {
    if (EVEN || base + c + 8 <= total) {
      v.load(p + base + c);
    } else {  // (the end of the tensor)
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = base + c + i < total ? float(p[base + c + i]) : 0.f;
      v.from_float(f);
    }
  }
  __device__ __forceinline__ void mask(float (&f)[8], int c) const {
    if (!whole(c)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i >= 0 && c + i < D ? f[i] : 0.f;
    }
  }
  __device__ __forceinline__ void store(const Vec8<T>& v, T* p, int c) const {
    if (whole(c)) {
      v.store(p + base + c);
    } else {
      float f[8];
      v.to_float(f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i >= 0 && c + i < D) p[base + c + i] = T(f[i]);
    }
  }
  __device__ __forceinline__ void weight(float (&f)[8], const T* w, int c) const {
    if (EVEN) {
      Vec8<T> v;
      v.load(w + c);
      v.to_float(f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i >= 0 && c + i < D ? float(w[c + i]) : 0.f;
    }
  }
  __device__ __forceinline__ void store_e4m3(const float (&f)[8], uint8_t* p, int c) const {  // (satfinite: what rounding puts a hair above 448 is 448)
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    if (whole(c)) {
      *reinterpret_cast<uint2*>(p + base + c) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i >= 0 && c + i < D) p[base + c + i] = (uint8_t)(q[i / 2] >> (8 * (i & 1)));
    }
  }
};
// vectors that a row may touch
static inline int row_vectors(int D) { return D % 8 == 0 ? D / 8 : (D + 14) / 8; }

struct AddNormOut {
  void *h, *y;  // h: null where there is no residual; y: null where only q is wanted
  float* rstd;
  uint8_t* q;  // null: no 8-bit result
  float* scale;
};

// block_sum, and the largest of the block's values with it (bits of magnitudes: a NaN is larger than everything); ``red``, ``red_top``: 32 words each
__device__ __forceinline__ float block_sum_top(float v, uint32_t& top, float* red, uint32_t* red_top) {
  v = warp_sum(v);
  top = __reduce_max_sync(0xffffffffu, top);
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
  __syncthreads();
  if (l == 0) {
    red[w] = v;
    red_top[w] = top;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, l < nw ? red_top[l] : 0u);
  return warp_sum(l < nw ? red[l] : 0.f);
}

// A warp (WARP_ROWS) or a block has a row, each thread up to NP vectors.
// In 8 bits 1 / rms cancels: with m = max |h w|, y / (max |y| / 448) = h w 448 / m, where h w of two bf16 is exact in fp32.  So q takes one rounded factor, is
// nearer to the formula than y / s would be (a third of the values that round the other way), and m is found in the same reduction as the sum of squares.
// Where h w or 448 / m may be no fp32 number (m below 2^-100, zeros among them, infinite or NaN) the row is gone through once more, with h r w.
// (Four blocks of eight warps to an SM where the compiler would take a few registers too many for them.)
template <typename T, bool EVEN, int NP, bool WARP_ROWS, bool FP8>
__global__ void __launch_bounds__(WARP_ROWS ? 256 : 1024, FP8 && WARP_ROWS && sizeof(T) == 2 && NP <= (EVEN ? 2 : 1) ? 4 : 0) add_rms_norm_kernel(const T* x, const T* res, const T* w, const AddNormOut o, long long rows, int D,
                                                                              float eps) {
  after_previous();
  __shared__ float red[32];
  __shared__ uint32_t red_top[32];
  const int tpr = WARP_ROWS ? 32 : blockDim.x;
  const int t = WARP_ROWS ? (threadIdx.x & 31) : threadIdx.x;
  const long long step = WARP_ROWS ? gridDim.x * (long long)(blockDim.x >> 5) : gridDim.x;
  for (long long row = WARP_ROWS ? blockIdx.x * (long long)(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; row < rows; row += step) {
    const Row<T, EVEN> at(row, rows, D);
    Vec8<T> v[NP], u[NP];
    float ss = 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = at.col(t + j * tpr);
      if (c < D) {
        at.load(v[j], x, c);
        if (res != nullptr) at.load(u[j], res, c);
      }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = at.col(t + j * tpr);
      if (c < D) {
        float f[8];
        v[j].to_float(f);
        if (res != nullptr) {
          float g[8];
          u[j].to_float(g);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] += g[i];
          v[j].from_float(f);  // h as it is stored is what the norm is taken of
          at.store(v[j], reinterpret_cast<T*>(o.h), c);
          v[j].to_float(f);
        }
        at.mask(f, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += f[i] * f[i];
        if (FP8) {
          float g[8];
          at.weight(g, w, c);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i] * g[i]) & 0x7fffffffu);
        }
      }
    }
    if (!FP8) {
      ss = WARP_ROWS ? warp_sum(ss) : block_sum(ss, red);
    } else if (WARP_ROWS) {
      ss = warp_sum(ss);
      top = __reduce_max_sync(0xffffffffu, top);
    } else {
      ss = block_sum_top(ss, top, red, red_top);
    }
    const float r = rsqrtf(ss / D + eps);
    if (t == 0) o.rstd[row] = r;
    float k = 0.f;  // q = h w k
    bool coded = !FP8;
    if (FP8) {
      const float m = __uint_as_float(top), r8 = __frsqrt_rn(__fdiv_rn(ss, (float)D) + eps);
      if (m >= 0x1p-100f && m < INFINITY) {
        const float amax = m * r8;
        const bool tiny = amax < 0x1p-100f;
        k = tiny ? r8 : __fdiv_rn(448.f, m);
        if (t == 0) o.scale[row] = tiny ? 1.f : __fdiv_rn(amax, 448.f);
      } else {  // (all threads of the row; apart from the others, whom a factor more would cost registers: 8192 x 2048 codes only 27.7 -> 31 us)
        coded = true;
        top = 0;
        auto each = [&](auto use) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const int c = at.col(t + j * tpr);
            if (c < D) {
              float f[8], g[8];
              v[j].to_float(f);
              at.mask(f, c);
              at.weight(g, w, c);
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = f[i] * r8 * g[i];
              use(f, c);
            }
          }
        };
        each([&](const float (&f)[8], int) {
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
        });
        if (WARP_ROWS) top = __reduce_max_sync(0xffffffffu, top);
        else block_sum_top(0.f, top, red, red_top);
        const float amax = __uint_as_float(top);
        const bool tiny = amax < 0x1p-100f;
        k = tiny ? 1.f : __fdiv_rn(448.f, amax);
        each([&](float (&f)[8], int c) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= k;
          at.store_e4m3(f, o.q, c);
        });
        if (t == 0) o.scale[row] = tiny ? 1.f : __fdiv_rn(amax, 448.f);
      }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = at.col(t + j * tpr);
      if (c < D) {
        float f[8], g[8];
        v[j].to_float(f);
        at.weight(g, w, c);
        if (!coded) {
          float q[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = f[i] * g[i] * k;
          at.store_e4m3(q, o.q, c);
        }
        if (!FP8 || o.y != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = f[i] * r * g[i];
          Vec8<T> ov;
          ov.from_float(f);
          at.store(ov, reinterpret_cast<T*>(o.y), c);
        }
      }
    }
  }
}

// Backward.  Blocks take rows in turn and keep their sums of dw in registers; each leaves one row of partial sums, which rms_dw_kernel adds up in order: the
// same result every time.  No power of r is formed: rows of any size that the forward pass takes have a gradient (r^3 would be no fp32 number from rms 2e12 on).  Where rows begin anywhere, the number of blocks is a multiple of 8, so that all rows of a block begin alike and a thread
// keeps its columns.
template <typename T, bool EVEN>
__device__ __forceinline__ void put_partial(const Row<T, EVEN>& at, float* part, const float (&dw)[8], int c) {
  float* p = part + (long long)blockIdx.x * at.D + c;
  if (EVEN) {
    reinterpret_cast<float4*>(p)[0] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(dw[4], dw[5], dw[6], dw[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i >= 0 && c + i < at.D) p[i] = dw[i];
  }
}

// For rows that the ring below does not hold: a row is read twice, the second time out of L2 (kept in registers it spills).
template <typename T, bool EVEN, int NP>
__global__ void __launch_bounds__(1024) add_rms_norm_bwd_kernel(const T* dy, const T* dh, const T* h, const T* w, const float* rstd, T* dx, float* part,
                                                                long long rows, int D) {
  after_previous();
  __shared__ float red[32];
  float dw[NP][8] = {};
  const float inv_d = 1.f / D;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const Row<T, EVEN> at(row, rows, D);
    const float r = rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = at.col(threadIdx.x + j * blockDim.x);
      if (c < D) {
        Vec8<T> hv, gv;
        at.load(hv, h, c);
        at.load(gv, dy, c);
        float hf[8], gf[8], wf[8];
        hv.to_float(hf);
        gv.to_float(gf);
        at.mask(hf, c);
        at.mask(gf, c);
        at.weight(wf, w, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float gh = gf[i] * hf[i];
          dw[j][i] = fmaf(gh, r, dw[j][i]);
          dot = fmaf(gh, wf[i], dot);
        }
      }
    }
    dot = block_sum(dot, red);
    const float mean = r * dot * inv_d;  // of g n
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int c = at.col(threadIdx.x + j * blockDim.x);
      if (c < D) {
        Vec8<T> hv, gv, ev;
        at.load(hv, h, c);
        at.load(gv, dy, c);
        float hf[8], gf[8], ef[8] = {}, wf[8];
        if (dh != nullptr) {
          at.load(ev, dh, c);
          ev.to_float(ef);
        }
        hv.to_float(hf);
        gv.to_float(gf);
        at.weight(wf, w, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) ef[i] = fmaf(r, fmaf(-(hf[i] * r), mean, gf[i] * wf[i]), ef[i]);
        ev.from_float(ef);
        at.store(ev, dx, c);
      }
    }
  }
  const Row<T, EVEN> at(blockIdx.x, rows, D);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int c = at.col(threadIdx.x + j * blockDim.x);
    if (c < D) put_partial(at, part, dw[j], c);
  }
}

// Where two or three rows of all three operands fit into shared memory: the rows arrive as bulk copies, issued ST - 1 steps ahead by one thread, so what is
// under way costs no registers and does not wait for the reduction (the ring of the plain norm's backward kernel, elementwise.cu, with a third operand).
// One block barrier a step: the sums of consecutive steps sit in alternating slots, and a stage is refilled behind the barrier of the step after its own,
// which every thread reaches when it has read the stage for the last time.  Waits are bounded: if a stage never arrives, the block records that in ``status`` and stops.
// A row that begins anywhere is copied with the vectors it touches; the last few elements of the tensor, where they are no whole vector, are read from
// memory.
__host__ __device__ inline int bwd_slot_bytes(int D, int elem) { return (D % 8 == 0 ? D : (D + 14) / 8 * 8) * elem; }
__host__ __device__ inline int bwd_ring_bytes(int D, int elem, int stages) { return stages * 3 * bwd_slot_bytes(D, elem) + 128; }
template <typename T, bool EVEN, int NVEC, int THREADS, int ST>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? (NVEC == 1 ? 4 : 3) : 1)
add_rms_norm_bwd_bulk_kernel(const T* dy, const T* dh, const T* h, const T* w, const float* rstd, T* dx, float* part, long long rows, int D, uint32_t* status) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[ST];
  __shared__ float red[2][THREADS / 32];
  __shared__ uint32_t abort_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~uintptr_t(127));
  const int slot = bwd_slot_bytes(D, (int)sizeof(T));
  volatile uint32_t* abort_flag = &abort_word;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&bars[s], 1);
    abort_word = 0;
    mbar_fence_init();
  }
  __syncthreads();
  after_previous();
  const long long step = gridDim.x, first = blockIdx.x;
  // elements of the row's vectors that a copy brings: all but those past the tensor's last whole 16 bytes
  auto copied = [&](const Row<T, EVEN>& at) -> int {
    if (EVEN) return D;
    const long long end = min((at.base + D + 7) / 8 * 8, at.total * (long long)sizeof(T) / 16 * (16 / (long long)sizeof(T)));
    return (int)(end - (at.base - at.lead));
  };
  auto issue = [&](long long it) {  // one thread: start the copies of this block's step ``it``
    const long long row = first + it * step;
    if (row >= rows) return;
    const Row<T, EVEN> at(row, rows, D);
    const int st = (int)(it % ST);
    const long long from = at.base - at.lead;
    const uint32_t bytes = (uint32_t)max(copied(at), 0) * (uint32_t)sizeof(T);
    uint8_t* to = smem + 3 * st * slot;
    mbar_expect_tx(&bars[st], (dh != nullptr ? 3u : 2u) * bytes);
    if (bytes == 0) return;
    bulk_load(to, h + from, bytes, &bars[st]);
    bulk_load(to + slot, dy + from, bytes, &bars[st]);
    if (dh != nullptr) bulk_load(to + 2 * slot, dh + from, bytes, &bars[st]);
  };
  if (threadIdx.x == 0)
    for (int it = 0; it < ST - 1; ++it) issue(it);
  const Row<T, EVEN> mine(first, rows, D);  // (all rows of the block begin like its first)
  Vec8<T> wv[EVEN ? NVEC : 1];
  float wo[EVEN ? 1 : NVEC][8];
  float dw[NVEC][8];
  int col[NVEC];
#pragma unroll
  for (int j = 0; j < NVEC; ++j) {
    col[j] = mine.col(threadIdx.x + j * THREADS);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
    if (col[j] < D) {
      if (EVEN) wv[EVEN ? j : 0].load(w + col[j]);
      else mine.weight(wo[EVEN ? 0 : j], w, col[j]);
    }
  }
  auto weight = [&](float (&f)[8], int j) {
    if (EVEN) {
      wv[EVEN ? j : 0].to_float(f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = wo[EVEN ? 0 : j][i];
    }
  };
  const float inv_d = 1.f / D;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long it = 0;
  float r_next = first < rows ? rstd[first] : 0.f;
  for (long long row = first; row < rows; row += step, ++it) {
    const Row<T, EVEN> at(row, rows, D);
    const int st = (int)(it % ST);
    const float r = r_next;
    if (row + step < rows) r_next = rstd[row + step];
    if (!mbar_wait(&bars[st], (uint32_t)((it / ST) & 1), abort_flag)) {
      atomicCAS(status, 0u, (uint32_t)ST_TIMEOUT_FULL);
      *abort_flag = 1;
    }
    const uint8_t* in = smem + 3 * st * slot;
    const int have = copied(at) - at.lead;  // columns that the copies brought
    auto read = [&](Vec8<T>& v, int operand, const T* p, int c) {
      if (EVEN || c + 8 <= have) v.load(reinterpret_cast<const T*>(in + operand * slot) + at.lead + c);
      else at.load(v, p, c);
    };
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NVEC; ++j) {
      if (col[j] < D) {
        Vec8<T> hv, gv;
        read(hv, 0, h, col[j]);
        read(gv, 1, dy, col[j]);
        float hf[8], gf[8], wf[8];
        hv.to_float(hf);
        gv.to_float(gf);
        at.mask(hf, col[j]);
        at.mask(gf, col[j]);
        weight(wf, j);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float gh = gf[i] * hf[i];
          dw[j][i] = fmaf(gh, r, dw[j][i]);
          dot = fmaf(gh, wf[i], dot);
        }
      }
    }
    dot = warp_sum(dot);
    if (THREADS > 32) {
      if (lane == 0) red[it & 1][warp] = dot;
      __syncthreads();
      dot = 0.f;
#pragma unroll
      for (int k = 0; k < THREADS / 32; ++k) dot += red[it & 1][k];
    } else {
      __syncwarp();
    }
    if (*abort_flag) {  // (set before the barrier, so every thread leaves here; the copies that are still under way are waited for, with the same limit)
      volatile uint32_t none = 0;
      for (long long k = it; threadIdx.x == 0 && k < it + ST - 1 && first + k * step < rows; ++k) mbar_wait(&bars[k % ST], (uint32_t)((k / ST) & 1), &none);
      break;
    }
    if (threadIdx.x == 0) issue(it + ST - 1);
    const float mean = r * dot * inv_d;  // of g n
#pragma unroll
    for (int j = 0; j < NVEC; ++j) {
      if (col[j] < D) {
        Vec8<T> hv, gv, ev;
        read(hv, 0, h, col[j]);
        read(gv, 1, dy, col[j]);
        float hf[8], gf[8], ef[8] = {}, wf[8];
        if (dh != nullptr) {
          read(ev, 2, dh, col[j]);
          ev.to_float(ef);
        }
        hv.to_float(hf);
        gv.to_float(gf);
        weight(wf, j);
#pragma unroll
        for (int i = 0; i < 8; ++i) ef[i] = fmaf(r, fmaf(-(hf[i] * r), mean, gf[i] * wf[i]), ef[i]);
        ev.from_float(ef);
        at.store(ev, dx, col[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NVEC; ++j)
    if (col[j] < D) put_partial(mine, part, dw[j], col[j]);
}

constexpr int ADD_NORM_MAX = 32768;  // columns: 1024 threads with 32 elements each

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

struct BwdPlan {
  int threads, np, grid, stages, smem;  // vectors of a thread, stages of the ring (0: none)
};
// The ring: a warp per row up to 32 vectors, a vector to a thread up to 256 threads, then two, then 512 threads; blocks as shared memory holds, up to 1024
// threads of an SM (768 in small blocks, which leave more partial rows: 8192 x 1024 18.0 -> 19.0 us with 1024, x 2048 32 -> 28, x 4096 50.2 -> 48.5).  At least four rows to a block where there are enough, so that few rows do not leave as many partial rows of dw.
static BwdPlan bwd_plan(long long rows, int D, int elem, int num_sms) {
  BwdPlan p{};
  const int vecs = row_vectors(D), room = 220 * 1024;
  const bool ring = vecs <= 2048;  // (512 threads with four vectors)
  p.stages = ring && bwd_ring_bytes(D, elem, 3) <= room ? 3 : ring && bwd_ring_bytes(D, elem, 2) <= room ? 2 : 0;
  int per_sm = 1;
  if (p.stages) {
    p.threads = vecs <= 32 ? 32 : vecs <= 64 ? 64 : vecs <= 128 ? 128 : vecs <= 512 ? 256 : 512;
    const int np = (vecs + p.threads - 1) / p.threads;
    p.np = np <= 2 ? np : 4;
    p.smem = bwd_ring_bytes(D, elem, p.stages);
    // (a block takes 1024 bytes more, and its barriers)
    const int by_smem = 228 * 1024 / (p.smem + 1536), by_threads = p.threads == 32 ? 16 : (p.threads < 256 ? 768 : 1024) / p.threads;
    per_sm = by_smem < 1 ? 1 : by_smem < by_threads ? by_smem : by_threads;
    // Shared memory that one block more would not find: where registers leave room for it, the blocks that come early (launch.cuh) gather on a few SMs (8192 x 2048
    // bf16 33 -> 27 us, x 1024 18 -> 16).  Not for rows that begin anywhere, whose weights are read one by one through what is left as cache (8192 x 249 13.2 -> 15.1).
    const int alone = 228 * 1024 / (per_sm + 1) - 1024;
    if (D % 8 == 0 && p.smem < alone && alone <= room) p.smem = alone;
  } else {
    p.threads = 1024;
    p.np = D % 8 == 0 ? 4 : 5;  // (a row of 32767 elements may touch 4097 vectors)
  }
  const long long cap = (long long)num_sms * per_sm, quarter = (rows + 3) / 4, least = rows < num_sms ? rows : num_sms;
  long long g = quarter < cap ? quarter : cap;
  if (g < least) g = least;
  p.grid = (int)(D % 8 == 0 ? g : (g + 7) / 8 * 8);  // (blocks without rows leave zeros)
  return p;
}

template <typename T, bool EVEN>
static cudaError_t launch_fwd(const void* x, const void* res, const void* w, const AddNormOut& o, long long rows, int D, float eps, cudaStream_t st) {
  const bool fp8 = o.q != nullptr;
  auto launch = [&](auto kern, unsigned grid, int threads) {
    return launch_after(kern, grid, threads, 0, st, (const T*)x, (const T*)res, (const T*)w, o, rows, D, eps);
  };
#define APB_ADD_NORM(NP, WARP, GRID, THREADS) \
  return fp8 ? launch(add_rms_norm_kernel<T, EVEN, NP, WARP, true>, GRID, THREADS) : launch(add_rms_norm_kernel<T, EVEN, NP, WARP, false>, GRID, THREADS)
  const int vecs = row_vectors(D);
  if (vecs <= 128) {  // a warp to a row, eight rows a block
    const unsigned grid = (unsigned)((rows + 7) / 8);
    if (vecs <= 32) APB_ADD_NORM(1, true, grid, 256);
    if (vecs <= 64) APB_ADD_NORM(2, true, grid, 256);
    APB_ADD_NORM(4, true, grid, 256);
  }
  int threads = 256;
  while (threads * 4 < vecs && threads < 1024) threads *= 2;
  const int np = (vecs + threads - 1) / threads;
  const unsigned grid = (unsigned)rows;
  if (np == 1) APB_ADD_NORM(1, false, grid, threads);
  if (np == 2) APB_ADD_NORM(2, false, grid, threads);
  if (EVEN || np <= 4) APB_ADD_NORM(4, false, grid, threads);
  APB_ADD_NORM((EVEN ? 4 : 5), false, grid, threads);  // (see bwd_plan)
#undef APB_ADD_NORM
}

template <typename T, bool EVEN>
static cudaError_t launch_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx, void* dw, float* part,
                              long long rows, int D, int num_sms, cudaStream_t st, uint32_t* status, int dw_fp32) {
  const BwdPlan p = bwd_plan(rows, D, (int)sizeof(T), num_sms);
  auto launch = [&](auto kern, auto... more) {
    if (p.smem && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem) != cudaSuccess) return cudaErrorInvalidValue;
    return launch_after(kern, p.grid, p.threads, p.smem, st, (const T*)dy, (const T*)dh, (const T*)h, (const T*)w, rstd, (T*)dx, part, rows, D, more...);
  };
  cudaError_t e = cudaErrorInvalidValue;
#define APB_RING(NV, TH, ST) \
  if (p.np == NV && p.threads == TH && p.stages == ST) e = launch(add_rms_norm_bwd_bulk_kernel<T, EVEN, NV, TH, ST>, status)
  if (p.stages) {
    APB_RING(1, 32, 3);
    APB_RING(1, 64, 3);
    APB_RING(1, 128, 3);
    APB_RING(1, 256, 3);
    APB_RING(2, 256, 3);
    APB_RING(2, 512, 3);
    APB_RING(4, 512, 2);
    if constexpr (sizeof(T) == 2) {  // (which rows need two stages: bf16 from about 12500 columns on, fp32 from 6250)
      APB_RING(4, 512, 3);
    } else {
      APB_RING(2, 512, 2);
    }
  } else {
    e = launch(add_rms_norm_bwd_kernel<T, EVEN, EVEN ? 4 : 5>);
  }
#undef APB_RING
  if (e != cudaSuccess) return e;
  const unsigned grid = (unsigned)((D + 31) / 32);
  if (dw_fp32) return launch_after(rms_dw_kernel<float>, grid, 1024, 0, st, (const float*)part, (float*)dw, p.grid, D);
  return launch_after(rms_dw_kernel<T>, grid, 1024, 0, st, (const float*)part, (T*)dw, p.grid, D);
}

}  // namespace apb

using namespace apb;

// 16-byte bases.  Returns 0, or an argument / launch error (nothing launched).
extern "C" int apb_add_rms_norm(const void* x, const void* res, const void* w, void* h, void* y, float* rstd, void* q, float* scale, long long rows, int D,
                                float eps, int is_bf16, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (D <= 0 || D > ADD_NORM_MAX || rows > 0x7fffffffll || (res != nullptr && h == nullptr) || (y == nullptr && q == nullptr)) return 3;
  for (const void* p : {x, res, w, (const void*)h, (const void*)y, (const void*)q})
    if (off16(p)) return 3;
  const AddNormOut o{h, y, rstd, (uint8_t*)q, scale};
  auto go = [&](auto even) {
    constexpr bool E = decltype(even)::value;
    return is_bf16 ? launch_fwd<bf16, E>(x, res, w, o, rows, D, eps, st) : launch_fwd<float, E>(x, res, w, o, rows, D, eps, st);
  };
  const cudaError_t e = D % 8 == 0 ? go(std::true_type{}) : go(std::false_type{});
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4;
}

// floats of workspace: a partial row of dw per block
extern "C" long long apb_add_rms_norm_bwd_workspace(long long rows, int D, int is_bf16, int num_sms) {
  return rows <= 0 || D <= 0 ? 0 : (long long)bwd_plan(rows, D, is_bf16 ? 2 : 4, num_sms).grid * D;
}
// ``status``: a word of device memory, which a wait that runs out is recorded in.  ``dw_fp32``: dw in fp32 (its sums as they are), else in the operands' type.
extern "C" int apb_add_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* w, const float* rstd, void* dx, void* dw, float* part,
                                    long long rows, int D, int is_bf16, int num_sms, cudaStream_t st, uint32_t* status,
                                    int dw_fp32) {
  if (rows <= 0 || D <= 0 || D > ADD_NORM_MAX || status == nullptr) return 3;
  for (const void* p : {dy, dh, h, w, (const void*)dx})
    if (off16(p)) return 3;
  auto go = [&](auto even) {
    constexpr bool E = decltype(even)::value;
    return is_bf16 ? launch_bwd<bf16, E>(dy, dh, h, w, rstd, dx, dw, part, rows, D, num_sms, st, status, dw_fp32)
                   : launch_bwd<float, E>(dy, dh, h, w, rstd, dx, dw, part, rows, D, num_sms, st, status, dw_fp32);
  };
  const cudaError_t e = D % 8 == 0 ? go(std::true_type{}) : go(std::false_type{});
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 4;
}
