// 16-bit operand times the values of an MXFP4 matrix, sm_100a: the gradient of a 4-bit product with respect to its activations.
//
//   C[g][M, K] = A[g][M, N] * values(B[g][N, K])      A bf16, B codes and scales with blocks along K, sums in fp32, C bf16 or fp32
//
// B is the weight as the forward product has it, so its values are written nowhere: a stage's codes (64 rows x 128 bytes) are turned into bf16 in shared
// memory, in the layout of an MN-major operand, and go from there to tcgen05.mma.  Against turning B into a bf16 matrix first that saves writing and reading
// it at 2 bytes a value (64 experts of 1408 x 2048: 740 MB), which is more than everything else of such a gradient over few rows.
//
// B takes the 128 rows of the MMA (twice: a tile has 256 columns of C), A's rows its N, up to 256 and a multiple of 16: an MMA's time is what it reads from
// shared memory, so that 160 rows cost 160 and not 256.  The two accumulators take all of TMEM, so that what is turned is used by as many rows as there may be.
// Measured: 64 experts of 1408 x 2048, 160 rows 88 us (0.67 PFLOP/s; 37 % of the tensor cores' cycles, 20 % of DRAM, 45 % of the issue slots), 1280 rows 448
// (1.05); the MMAs, whose operand of 128 rows is read again for every 16 of its columns, and the turning of codes wait for each other's slots.
//   warp 0: TMA producer (A, codes, scales) | warp 1: TMEM owner, MMAs | warps 2..9: codes to values, then the tile's epilogue
#include <algorithm>

#include "mx4.cuh"

namespace apb {

constexpr int MV_WARPS = 8, MV_THREADS = 64 + 32 * MV_WARPS;
constexpr int MV_BN = 64, MV_COLS = 256;  // rows of B in a stage, and columns of the tile
constexpr int MV_A = 256 * MV_BN * 2, MV_CODES = MV_BN * MX_ROW_BYTES, MV_SLOT = MV_BN * MV_COLS * 2;  // bytes of a stage: of A, of codes, of values
// Rings of A, of codes with their scales, and of values.  Codes come from memory, and a stage has few of them: their ring is longer, and runs ahead of A's.
constexpr int MV_A_RING = 3, MV_C_RING = 6, MV_V_RING = 2, MV_AHEAD = MV_C_RING - MV_A_RING;
constexpr int MV_SMEM = 1024 + MV_A_RING * MV_A + MV_C_RING * (MV_CODES + MX_SC_BYTES) + MV_V_RING * MV_SLOT + 256;
static_assert(MV_SMEM <= 227 * 1024, "shared memory of a CTA");

struct MxValuesParams {
  GemmParams p;  // M, N = columns of C, ldc, out_fp32, status
  int tiles, m_tiles, stages;  // stages: of 64 along the contraction
  int vec;                      // rows of C are whole 16 bytes
};

__device__ __forceinline__ uint32_t mx_prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// Four codes (the low 16 bits of ``w``) to two words of bf16 pairs: bytes of the magnitudes' high and low halves from tables of eight, the sign, interleaved.
// (With bit 3 of a selector set prmt repeats the sign of the byte: 0x80 for a positive code, 0xFF for a negative one.)
__device__ __forceinline__ void mx_four_bf16(uint32_t w, uint32_t magnitude, uint32_t& r0, uint32_t& r1) {
  const uint32_t sign = mx_prmt(0x80808080u, 0x80808080u, w) << 1;
  const uint32_t lo = mx_prmt(0xC0800000u, 0xC0804000u, magnitude), hi = mx_prmt(0x3F3F3F00u, 0x40404040u, magnitude) | (sign & 0x80808080u);
  r0 = mx_prmt(lo, hi, 0x5140);
  r1 = mx_prmt(lo, hi, 0x7362);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__global__ void __launch_bounds__(MV_THREADS, GEMM_MIN_CTAS)
gemm_mx4_values_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSB,
                       MxValuesParams q) {
  const GemmParams& p = q.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;                         // [ring] 256 rows of 128 bytes
  uint8_t* sB = sA + MV_A_RING * MV_A;        // [ring] codes: 64 rows of 128 bytes
  uint8_t* sV = sB + MV_C_RING * MV_CODES;    // [ring] values: four chunks of 64 columns, 64 rows of 128 bytes each
  uint8_t* sSc = sV + MV_V_RING * MV_SLOT;    // [ring of the codes] scales of 128 rows
  uint64_t* bars = reinterpret_cast<uint64_t*>(sSc + MV_C_RING * MX_SC_BYTES);
  uint64_t *a_full = bars, *a_empty = a_full + MV_A_RING, *c_full = a_empty + MV_A_RING, *c_empty = c_full + MV_C_RING, *turned = c_empty + MV_C_RING,
           *used = turned + MV_V_RING, *acc_full = used + MV_V_RING, *acc_free = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert((2 * (MV_A_RING + MV_C_RING + MV_V_RING) + 3) * 8 <= 256, "barrier block");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MV_A_RING; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], 1);
    }
    for (int s = 0; s < MV_C_RING; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], MV_WARPS);
    }
    for (int s = 0; s < MV_V_RING; ++s) {
      mbar_init(&turned[s], MV_WARPS);
      mbar_init(&used[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_free, MV_WARPS);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_previous();

  auto fail = [&](uint32_t code) {
    atomicCAS(p.status, 0u, code);
    *abort_flag = 1;
  };
  // tile -> group, rows, columns; the row tiles of a column tile come one after the other: its codes are in L2 then
  auto place = [&](int t, int& grp, int& m0, int& col) {
    grp = p.div_tiles.div(t);
    const int r = t - grp * (int)p.div_tiles.d, tn = p.div_group.div(r);
    m0 = (r - tn * q.m_tiles) * 256;
    col = tn * MV_COLS;
  };
  if (warp == 0) {
    if (elect_one()) {
      struct At {  // a stage of this CTA's sequence
        int t, k, grp, m0, col;
        uint32_t it;
      };
      auto begin = [&](At& a) {
        if (a.t < q.tiles) place(a.t, a.grp, a.m0, a.col);
      };
      auto step = [&](At& a) {
        ++a.it;
        if (++a.k == q.stages) {
          a.k = 0;
          a.t += gridDim.x;
          begin(a);
        }
      };
      auto load_codes = [&](const At& c) {
        const uint32_t s = c.it % MV_C_RING;
        if (!mbar_wait(&c_empty[s], (c.it / MV_C_RING & 1) ^ 1, abort_flag)) return false;
        mbar_expect_tx(&c_full[s], MV_CODES + MX_SC_BYTES);
        tma_load_3d(sB + s * MV_CODES, &tmB, &c_full[s], c.col / 2, c.k * MV_BN, c.grp);
        tma_load_3d(sSc + s * MX_SC_BYTES, &tmSB, &c_full[s], c.col / MX_BK * (MX_SC_BYTES / 4), c.k * MV_BN / 128, c.grp);
        return true;
      };
      At a{(int)blockIdx.x, 0, 0, 0, 0, 0u};
      begin(a);
      At c = a;
      bool ok = true;
      while (a.t < q.tiles && ok) {
        while (c.t < q.tiles && c.it <= a.it + MV_AHEAD && ok) {
          ok = load_codes(c);
          step(c);
        }
        const uint32_t s = a.it % MV_A_RING;
        if (!ok || !mbar_wait(&a_empty[s], (a.it / MV_A_RING & 1) ^ 1, abort_flag)) {
          fail(ST_TIMEOUT_EMPTY);
          break;
        }
        const bool two = p.M - a.m0 > 128;
        mbar_expect_tx(&a_full[s], two ? MV_A : MV_A / 2);
        tma_load_3d(sA + s * MV_A, &tmA, &a_full[s], a.k * MV_BN, a.m0, a.grp);
        if (two) tma_load_3d(sA + s * MV_A + MV_A / 2, &tmA, &a_full[s], a.k * MV_BN, a.m0 + 128, a.grp);
        step(a);
      }
      let_next_in();
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t a_desc = make_smem_desc(smem_u32(sA), 16, 1024), v_desc = make_smem_desc(smem_u32(sV), CHUNK_BYTES, 1024);
      uint32_t it = 0, seq = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x, ++seq) {
        int grp, m0, col;
        place(t, grp, m0, col);
        const uint32_t idesc = make_idesc_bf16(128, (min(p.M - m0, 256) + 15) / 16 * 16, 1, 0);
        if (seq > 0 && !mbar_wait(acc_free, (seq - 1) & 1, abort_flag)) {
          fail(ST_TIMEOUT_TMEM_EMPTY);
          break;
        }
        tc_fence_after();
        for (int k = 0; k < q.stages; ++k, ++it) {
          const uint32_t s = it % MV_A_RING, v = it % MV_V_RING;
          if (!mbar_wait(&a_full[s], it / MV_A_RING & 1, abort_flag) || !mbar_wait(&turned[v], it / MV_V_RING & 1, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_FULL);
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < MV_BN / UMMA_K; ++kk) {
            const uint64_t ad = a_desc + desc_offset(s * MV_A + kk * UMMA_K * 2), vd = v_desc + desc_offset(v * MV_SLOT + kk * UMMA_K * 128);
            const uint32_t more = k > 0 || kk > 0 ? 1u : 0u;
            umma_f16(tmem, vd, ad, idesc, more);
            umma_f16(tmem + 256, vd + desc_offset(MV_SLOT / 2), ad, idesc, more);
          }
          umma_commit(&a_empty[s]);
          umma_commit(&used[v]);
        }
        if (ok) umma_commit(acc_full);
      }
    }
  } else {
    const int w = warp - 2, quarter = warp & 3, half = w >> 2;
    // A warp turns eight rows of a stage, a lane two blocks of 32 columns of one: eight lanes on eight rows, so that neither the swizzled codes nor the
    // values meet in a bank.
    const int row = w * 8 + (lane & 7), block = lane >> 3, swizzle = lane & 7;
    const uint32_t from = row * 128 + ((block ^ swizzle) << 4), from2 = row * 128 + (((block + 4) ^ swizzle) << 4);  // bytes of a stage's codes
    const uint32_t to = (block >> 1) * CHUNK_BYTES + row * 128, unit = ((block & 1) * 4) ^ swizzle;                   // and of its values
    uint32_t seq = 0, c_slot = 0, c_phase = 0, v_slot = 0, v_phase = 1;
    bool ok = true;
    for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x, ++seq) {
      int grp, m0, col;
      place(t, grp, m0, col);
      for (int k = 0; k < q.stages; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait(&c_full[c_slot], c_phase, abort_flag) && mbar_wait(&used[v_slot], v_phase, abort_flag));
        if (!ok) {
          fail(ST_TIMEOUT_FULL);
          break;
        }
        const uint8_t *codes = sB + c_slot * MV_CODES, *sc = sSc + c_slot * MX_SC_BYTES + mx_scale_at((k * MV_BN + row) & 127, block);
        uint8_t* values = sV + v_slot * MV_SLOT + to;
        const uint4 c[2] = {*reinterpret_cast<const uint4*>(codes + from), *reinterpret_cast<const uint4*>(codes + from2)};
        const uint32_t e[2] = {sc[0], sc[MX_SCALE_TILE]};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t scale = (e[i] == 255u ? 0x7FC0u : e[i] == 0u ? 0x0040u : e[i] << 7) * 0x10001u;
          const uint32_t x[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t magnitude = x[u] & 0x77777777u;
            uint32_t r[4];
            mx_four_bf16(x[u], magnitude, r[0], r[1]);
            mx_four_bf16(x[u] >> 16, magnitude >> 16, r[2], r[3]);
            *reinterpret_cast<uint4*>(values + i * 2 * CHUNK_BYTES + ((unit ^ u) << 4)) =
                make_uint4(mul_bf16x2(r[0], scale), mul_bf16x2(r[1], scale), mul_bf16x2(r[2], scale), mul_bf16x2(r[3], scale));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&turned[v_slot]);
          mbar_arrive(&c_empty[c_slot]);
        }
        if (++c_slot == MV_C_RING) c_slot = 0, c_phase ^= 1;
        if (++v_slot == MV_V_RING) v_slot = 0, v_phase ^= 1;
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full, seq & 1, abort_flag));
      if (!ok) {
        fail(ST_TIMEOUT_TMEM_FULL);
        break;
      }
      tc_fence_after();
      // A warp has 32 columns of C in its TMEM lanes, half of the warps in the one accumulator and half in the other; A's rows are TMEM columns.  Through the
      // values' ring, which is free until this warp and the others turn the next tile's first stage, they become rows of 256 columns again.
      const int rows = min(p.M - m0, 256), esz = p.out_fp32 ? 4 : 2, at_once = MV_V_RING * MV_SLOT / (MV_COLS * 4);
      const int columns = min(MV_COLS, p.N - col);
      uint8_t* C = reinterpret_cast<uint8_t*>(p.C) + (((long long)grp * p.M + m0) * p.ldc + col) * esz;
      for (int first = 0; first < rows; first += at_once) {
#pragma unroll 1
        for (int m = first; m < min(rows, first + at_once); m += 32) {
          uint32_t r[32];
          tmem_ld_32x32(tmem + (uint32_t(quarter * 32) << 16) + half * 256 + m, r);
          tmem_ld_wait_for(r);
          uint8_t* mine = sV + (m - first) * MV_COLS * esz + (128 * half + 32 * quarter + lane) * esz;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (p.out_fp32) *reinterpret_cast<uint32_t*>(mine + i * MV_COLS * 4) = r[i];
            else *reinterpret_cast<__nv_bfloat16*>(mine + i * MV_COLS * 2) = __float2bfloat16(__uint_as_float(r[i]));
          }
        }
        named_sync(1, 32 * MV_WARPS);
        const int here = min(at_once, rows - first);
        if (q.vec) {
          const int units = MV_COLS * esz / 16;
          for (int i = threadIdx.x - 64; i < here * units; i += 32 * MV_WARPS) {
            const int m = i / units, u = i - m * units;
            if (u * 16 < columns * esz)
              *reinterpret_cast<uint4*>(C + (first + m) * p.ldc * esz + u * 16) = *reinterpret_cast<const uint4*>(sV + (m * units + u) * 16);
          }
        } else {
          for (int i = threadIdx.x - 64; i < here * MV_COLS; i += 32 * MV_WARPS) {
            const int m = i / MV_COLS, u = i - m * MV_COLS;
            if (u >= columns) continue;
            uint8_t* dst = C + ((first + m) * p.ldc + u) * esz;
            if (p.out_fp32) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(sV + i * 4);
            else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(sV + i * 2);
          }
        }
        named_sync(1, 32 * MV_WARPS);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_free);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace apb

using namespace apb;

extern "C" int apb_gemm_get_reserved_sms();

// Whether this kernel is the better choice against the values as a matrix of their own and the 16-bit product: with few rows, where the matrix is most of
// what is moved, and tiles for every SM.  us, this / that: 64 experts of 1408 x 2048, 16 rows 69 / 147, 160 rows 88 / 165, 1280 rows 448 / 392; 16 of 2048 x
// 2048, 512 rows 73 / 84; one of 4096 x 4096, 2048 rows (128 tiles) 60 / 54, of 4096 x 14336, 1024 rows 116 / 104, of 14336 x 4096, 16 rows (16 tiles)
// 153 / 48.  Three slots of values for two, sixteen warps for eight change nothing: the MMAs, whose operand of 128 rows comes in 16 of its columns at a time, are
// the bound.
extern "C" int apb_gemm_mx4_values_takes(long long G, long long M, long long K, int num_sms) {
  return M <= 512 && G * ((M + 255) / 256) * ((K + MV_COLS - 1) / MV_COLS) >= num_sms;
}

// A [G, M, N] bf16 (N % 8 == 0), B codes [G, N, kp / 2] and SB, C [G, M, K]; all dense, 16-byte bases.
// Returns 0, or an argument / driver / launch error (nothing launched; 3: not this kernel's form).
extern "C" int apb_gemm_mx4_values(const void* A, const void* B, const void* SB, void* C, long long G, long long M, long long N, long long K, int out_fp32,
                                   uint32_t* status, int num_sms, cudaStream_t stream) {
  const long long kp = (K + 31) / 32 * 32;
  if (G < 0 || M < 0 || N < 0 || K < 0 || M >= 1ll << 30 || N >= 1ll << 30 || K >= 1ll << 30 || N % 8) return 3;
  if (G == 0 || M == 0 || K == 0) return 0;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(SB) | reinterpret_cast<uintptr_t>(C)) & 15) return 3;
  if (N == 0) return zero_result(C, G * M, K, K, out_fp32, stream);
  MxValuesParams q{};
  GemmParams& p = q.p;
  p.M = (int)M;
  p.N = (int)K;
  p.C = C;
  p.ldc = K;
  p.out_fp32 = out_fp32;
  p.status = status;
  q.m_tiles = (int)((M + 255) / 256);
  q.stages = (int)((N + MV_BN - 1) / MV_BN);
  q.vec = K * (out_fp32 ? 4 : 2) % 16 == 0;
  const long long n_tiles = (K + MV_COLS - 1) / MV_COLS, tiles = G * q.m_tiles * n_tiles;
  if (tiles >= 1ll << 30) return 3;
  q.tiles = (int)tiles;
  p.div_tiles = FastDiv((uint32_t)(q.m_tiles * n_tiles));
  p.div_group = FastDiv((uint32_t)q.m_tiles);
  CUtensorMap tmA, tmB, tmSB;
  int e = make_map_3d(&tmA, A, (uint64_t)N, (uint64_t)M, (uint64_t)G, (uint64_t)N, BM);
  if (!e) e = mx_map(&tmB, B, kp / 2, N, G, MX_ROW_BYTES, MV_BN, false);
  if (!e) e = mx_map(&tmSB, SB, (uint64_t)((kp + 127) / 128) * (MX_SCALE_TILE / 4), (N + 127) / 128, G, MX_SC_BYTES / 4, 1, true);
  if (e) return e;
  const int usable = std::max(1, num_sms - apb_gemm_get_reserved_sms());
  cudaFuncSetAttribute(gemm_mx4_values_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MV_SMEM);
  launch_after(gemm_mx4_values_kernel, (unsigned)std::min(q.tiles, usable), MV_THREADS, MV_SMEM, stream, tmA, tmB, tmSB, q);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
