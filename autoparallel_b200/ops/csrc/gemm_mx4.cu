// Products of MXFP4 matrices on the block-scaled tensor cores of sm_100a (formats and layout in ops/mx4_ops.py):
//
//   C[g][M, N] = A[g][M, K] * B[g][N, K]^T, both in 4 bits with a scale for 32 values along K; sums in fp32, C bf16 or fp32
//
// Persistent and warp-specialised like the 16-bit GEMM (gemm_core.cuh): TMA -> shared memory -> tcgen05.mma kind::mxf4 -> TMEM -> epilogue.  A stage is
// 256 values of K (rows of 128 bytes, 128-byte swizzle, as 64 bf16 would be) and the scale tiles that belong to them, which the MMA thread has copied
// to TMEM (tcgen05.cp) in front of the stage's MMAs.
//   warp 0: TMA producer | warp 1: TMEM owner, scale copies, MMAs | warps 2..9: epilogue, two per TMEM lane quarter, each half of the tile's columns
//
// Measured: 8192 x 14336 x 4096 162 us (5.9 PFLOP/s), 8192 x 4096 x 14336 151 (6.4), 8192 x 8192 x 8192 176 (6.2), 64 x 1280 x 1408 x 2048 107 (4.4 PFLOP/s, 3.9
// TB/s), 2048 x 4096 x 4096 17.4 (3.9).  Along K alone the rate is 7 PFLOP/s.  What is missing is the way from a tile's last MMA over the epilogue's shared
// columns to the next tile's first (some 1500 cycles of a tile, of 4096 of MMAs at K = 2048), and in long runs power.  Wider tiles with
// accumulators side by side (256 x 448 for a pair) have no such pause, but MMAs of fewer than 256 columns run below that rate: 174 us for the first, 123 for
// the fourth.
//
// TMEM: two accumulators of up to 256 columns and 24 columns of scales do not fit 512, so the accumulators overlap by 32 columns: 0 ... 255 and
// 224 ... 479, scales from 480 on.  The epilogue reads the shared columns first, and the next tile's MMAs start as soon as that is done.
#include <algorithm>

#include "mx4.cuh"

namespace apb {

constexpr int MX_ACC1 = 224, MX_SCALE_COL = 480;  // first columns of the second accumulator and of the scales
constexpr int MX_EPI_WARPS = 8, MX_GEMM_THREADS = 64 + 32 * MX_EPI_WARPS;
constexpr int MX_STAGING = MX_EPI_WARPS * 4096;
constexpr int MX_BAR_BYTES = 256;

// BT: tiles of 128 rows of B that a CTA stages (PAIR: one of the pair's two); its column tile is 128 * BT, the pair's 256
template <bool PAIR, int BT>
struct MxShape {
  static constexpr int SB_TILES = PAIR ? 2 : BT;  // every CTA needs the scales of all columns
  static constexpr int STAGE = MX_OP_BYTES * (1 + BT) + MX_SC_BYTES * (1 + SB_TILES);
  static constexpr int STAGES = (227 * 1024 - 1024 - MX_BAR_BYTES - MX_STAGING) / STAGE;
  static constexpr int SMEM = 1024 + STAGES * STAGE + MX_STAGING + MX_BAR_BYTES;
};

struct MxGemmParams {
  GemmParams p;  // M, N, C, ldc, out_fp32, status and the tile order
  int tiles, num_m, num_kb, k_steps;  // k_steps: MMAs of 64 along K
  int col_tile, store, grouped;
};
enum : int { MX_SCALAR = 0, MX_STAGED = 1, MX_DIRECT = 2 };

// 32 rows of 128 bytes from shared memory (16-byte units swizzled by the row) to rows that begin anywhere, of which ``rows`` and ``lim`` columns are in the
// matrix: a word a lane.  A bf16 row that begins in the middle of a word of memory has words of the second half of a lane's and the first of the next one's, and its
// first and last value by themselves; rows of an odd stride begin there every other time, so the even and the odd ones go by themselves, with the same
// addresses and conditions in all of them: two warps a scheduler wait for their own instructions here, and every one counts.  64 x 1280 x 1407 x 2048 133
// us this way (1408: 110), 175 with the conditions worked out in each row, 418 element by element; fp32 176, 182, 610 (141).
__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void mx_rows_anywhere(uint8_t* dst, long long step, const uint8_t* stg, int rows, int lim, bool fp32, int lane) {
  if (fp32) {
    const uint32_t from = smem_u32(stg) + lane * 4;
    uint8_t* at = dst + 4 * lane;
    if (lane >= lim) rows = 0;
#pragma unroll 1
    for (int b = 0; b < 32; b += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = ld_shared((from ^ (j << 4)) + (b + j) * 128);
#pragma unroll
      for (int j = 0; j < 8; ++j, at += step)
        if (b + j < rows) *reinterpret_cast<uint32_t*>(at) = w[j];
    }
  } else {
#pragma unroll 1
    for (int c = 0; c < 2; ++c, dst += step) {
      const uint32_t from = smem_u32(stg) + c * 128 + ((((lane >> 2) ^ c) << 4) | (lane & 3) * 4);
      const bool odd = (reinterpret_cast<uintptr_t>(dst) & 2) != 0;  // (in all lanes)
      const int e = 2 * lane + odd;                                  // first value of the lane's word
      const bool word = e + 1 < lim, tail = e + 1 == lim, head = odd && lane == 0;
      uint8_t* at = dst + 2 * e;
#pragma unroll 1
      for (int b = 0; b < 32; b += 8) {
        uint32_t w[4], own[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = own[j] = ld_shared((from ^ (j << 5)) + (b + 2 * j) * 128);
        if (odd) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(own[j], __shfl_down_sync(0xffffffffu, own[j], 1), 16);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j, at += 2 * step) {
          const bool in = b + 2 * j + c < rows;
          if (in && word) *reinterpret_cast<uint32_t*>(at) = w[j];
          if (in && tail) *reinterpret_cast<uint16_t*>(at) = (uint16_t)w[j];
          if (in && head) *reinterpret_cast<uint16_t*>(at - 2) = (uint16_t)own[j];
        }
      }
    }
  }
  __syncwarp();  // (together to the next load from TMEM)
}

// The epilogue where rows are no whole sectors (mx_store_direct where they are), 64 columns at a time: through shared memory in 16-byte pieces of whole
// 128-byte lines, or word by word.  64 x 1280 x 1408 x 256 66 us this way, 55 straight from registers.
template <typename Release>
__device__ __forceinline__ void mx_store_staged(const MxGemmParams& q, uint8_t* C, uint8_t* stg, uint32_t taddr, int row0, int n0, int ncols, bool down,
                                                int lane, Release release) {
  const GemmParams& p = q.p;
  const int esz = p.out_fp32 ? 4 : 2;
  const int chunks = row0 < p.M ? (min(ncols, p.N - n0) + 63) / 64 : 0;
  const bool early = chunks > 0 && !(down && chunks * 64 < ncols);
  if (!early) release();
#pragma unroll 1
  for (int i = 0; i < chunks; ++i) {
    const int c = (down ? chunks - 1 - i : i) * 64;
    uint32_t r[2][32];
    tmem_ld_32x32(taddr + c, r[0]);
    tmem_ld_32x32(taddr + c + 32, r[1]);
    tmem_ld_wait_for(r[0]);
    tmem_ld_wait_for(r[1]);
    if (early && i == 0) release();
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // fp32: 32 columns at a time; bf16: all 64 in the first
      if (h == 1 && !p.out_fp32) break;
      uint4 v[8];
      if (p.out_fp32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = make_uint4(r[h][4 * j], r[h][4 * j + 1], r[h][4 * j + 2], r[h][4 * j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t* x = r[j >> 2] + 8 * (j & 3);
          v[j] = make_uint4(pack_bf16(__uint_as_float(x[0]), __uint_as_float(x[1])), pack_bf16(__uint_as_float(x[2]), __uint_as_float(x[3])),
                            pack_bf16(__uint_as_float(x[4]), __uint_as_float(x[5])), pack_bf16(__uint_as_float(x[6]), __uint_as_float(x[7])));
        }
      }
      __syncwarp();  // the block before has been read out
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = v[j];
      __syncwarp();
      const int col0 = n0 + c + 32 * h;  // of the 128 bytes
      if (q.store == MX_STAGED) {
        const int unit = lane & 7, sub = lane >> 3, col = col0 + unit * (16 / esz);
#pragma unroll 4
        for (int j = 0; j < 8; ++j) {
          const int row = 4 * j + sub;
          const uint4 x = *reinterpret_cast<const uint4*>(stg + row * 128 + ((unit ^ (row & 7)) << 4));
          if (col < p.N && row0 + row < p.M) *reinterpret_cast<uint4*>(C + ((row0 + row) * p.ldc + col) * esz) = x;
        }
      } else {
        mx_rows_anywhere(C + (row0 * p.ldc + col0) * esz, p.ldc * esz, stg, min(32, p.M - row0), min(128 / esz, p.N - col0), p.out_fp32, lane);
      }
    }
  }
}

template <bool PAIR, int BT>
__device__ __forceinline__ void mx_gemm_cta(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmSA, const CUtensorMap& tmSB,
                                            const MxGemmParams& q, uint8_t* smem_raw) {
  using S = MxShape<PAIR, BT>;
  constexpr int ST = S::STAGES, TM = PAIR ? 256 : 128;
  constexpr int A_AT = 0, B_AT = MX_OP_BYTES, OP_STAGE = MX_OP_BYTES * (1 + BT), SC_STAGE = S::STAGE - OP_STAGE;
  const GemmParams& p = q.p;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // operands of all stages first (1024-byte atoms), then the scales
  uint8_t* ops = smem;
  uint8_t* scs = smem + ST * OP_STAGE;
  uint8_t* staging = smem + ST * S::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + MX_STAGING);
  uint64_t* full = bars;               // [ST]  PAIR: the even CTA's are used
  uint64_t* empty = bars + ST;         // [ST]
  uint64_t* acc_full = bars + 2 * ST;  // [2]
  uint64_t* go = bars + 2 * ST + 2;    // the columns that two accumulators share have been read; one arrival per epilogue warp, PAIR: of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * ST + 3);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert((2 * ST + 4) * 8 <= MX_BAR_BYTES, "barrier block");
  const uint32_t half = PAIR ? cluster_ctarank() : 0u;  // 0: issues the MMAs, owns the shared barriers
  const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, num_units = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(go, (PAIR ? 2 : 1) * MX_EPI_WARPS);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_previous();

  auto fail = [&](uint32_t code) {
    atomicCAS(p.status, 0u, code);
    *abort_flag = 1;
  };
  // columns of a tile's MMAs: a wide one with 128 columns or fewer takes half of them
  auto width = [&](int col) { return q.col_tile > 128 && p.N - col <= 128 ? 128 : q.col_tile; };
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      const uint32_t full_pair = PAIR ? map_to_cta(full, 0) : 0u;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = unit; t < q.tiles && ok; t += num_units) {
        int grp, tm, tn;
        plain_tile(p, q.num_m, q.grouped, t, grp, tm, tn);
        const int m0 = tm * TM + (int)half * 128, col = tn * q.col_tile;
        const int n0 = col + (PAIR ? (int)half * width(col) / 2 : 0);  // rows of B that this CTA stages
        for (int kb = 0; kb < q.num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_EMPTY);
            break;
          }
          uint8_t *op = ops + stage * OP_STAGE, *sc = scs + stage * SC_STAGE;
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
            if (PAIR) tma_load_3d_pair(dst, map, full_pair + stage * 8, x, y, grp);
            else tma_load_3d(dst, map, &full[stage], x, y, grp);
          };
          if (half == 0) mbar_expect_tx(&full[stage], (PAIR ? 2 : 1) * S::STAGE);
          load(op + A_AT, &tmA, kb * MX_ROW_BYTES, m0);
          load(op + B_AT, &tmB, kb * MX_ROW_BYTES, n0);
          load(sc, &tmSA, kb * (MX_SC_BYTES / 4), m0 / 128);
          load(sc + MX_SC_BYTES, &tmSB, kb * (MX_SC_BYTES / 4), col / 128);
          if (++stage == ST) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      let_next_in();
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ scale copies and MMAs
    if (half == 0 && elect_one()) {
      const uint64_t a_desc = make_smem_desc(smem_u32(ops + A_AT), 16, 1024), b_desc = make_smem_desc(smem_u32(ops + B_AT), 16, 1024);
      const uint64_t sa_desc = make_scale_desc(smem_u32(scs)), sb_desc = make_scale_desc(smem_u32(scs + MX_SC_BYTES));
      const uint32_t empty_even = PAIR ? map_to_cta(empty, 0) : 0u, empty_odd = PAIR ? map_to_cta(empty, 1) : 0u;
      const uint32_t sa_tmem = tmem + MX_SCALE_COL, sb_tmem = sa_tmem + 4 * MX_STAGE_TILES;
      int stage = 0;
      uint32_t phase = 0, seq = 0;
      bool ok = true;
      for (int t = unit; t < q.tiles && ok; t += num_units, ++seq) {
        if (seq > 0 && !mbar_wait(go, (seq - 1) & 1u, abort_flag)) {
          fail(ST_TIMEOUT_TMEM_EMPTY);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem + (seq & 1u) * MX_ACC1;
        int grp, tm, tn;
        plain_tile(p, q.num_m, q.grouped, t, grp, tm, tn);
        const uint32_t idesc[2] = {make_idesc_mx4(TM, width(tn * q.col_tile), 0), make_idesc_mx4(TM, width(tn * q.col_tile), 2)};
        for (int kb = 0; kb < q.num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_FULL);
            break;
          }
          tc_fence_after();
          auto copy = [&](uint32_t taddr, uint64_t desc) {
            if (PAIR) tmem_copy_scales_pair(taddr, desc);
            else tmem_copy_scales(taddr, desc);
          };
          const int steps = min(MX_BK / 64, q.k_steps - kb * (MX_BK / 64));
#pragma unroll
          for (int a = 0; a < MX_STAGE_TILES; ++a) {  // (the tiles of a row group lie after each other; a column of scales for 32 rows)
            copy(sa_tmem + 4 * a, sa_desc + desc_offset(stage * SC_STAGE + a * MX_SCALE_TILE));
#pragma unroll
            for (int b = 0; b < S::SB_TILES; ++b)
              copy(sb_tmem + 4 * (a * S::SB_TILES + b), sb_desc + desc_offset(stage * SC_STAGE + b * MX_SC_BYTES + a * MX_SCALE_TILE));
          }
          const uint64_t ad = a_desc + desc_offset(stage * OP_STAGE), bd = b_desc + desc_offset(stage * OP_STAGE);
#pragma unroll
          for (int s = 0; s < MX_BK / 64; ++s) {
            if (s >= steps) break;
            const uint32_t sa = sa_tmem + 4 * (s / 2), sb = sb_tmem + 4 * S::SB_TILES * (s / 2);
            const uint32_t more = kb > 0 || s > 0 ? 1u : 0u;
            if (PAIR) umma_mx4_pair(d_tmem, ad + desc_offset(32 * s), bd + desc_offset(32 * s), idesc[s & 1], sa, sb, more);
            else umma_mx4(d_tmem, ad + desc_offset(32 * s), bd + desc_offset(32 * s), idesc[s & 1], sa, sb, more);
          }
          if (PAIR) {
            umma_commit_pair(empty_even + stage * 8);
            umma_commit_pair(empty_odd + stage * 8);
          } else {
            umma_commit(&empty[stage]);
          }
          if (++stage == ST) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (PAIR) {
          umma_commit_pair(map_to_cta(&acc_full[seq & 1u], 0));
          umma_commit_pair(map_to_cta(&acc_full[seq & 1u], 1));
        } else {
          umma_commit(&acc_full[seq & 1u]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    const uint32_t go_even = PAIR ? map_to_cta(go, 0) : 0u;
    const int esz = p.out_fp32 ? 4 : 2;
    uint32_t seq = 0;
    for (int t = unit; t < q.tiles; t += num_units, ++seq) {
      int grp, tm, tn;
      plain_tile(p, q.num_m, q.grouped, t, grp, tm, tn);
      const uint32_t buf = seq & 1u;
      const int cols = width(tn * q.col_tile) / 2;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster_plain(go_even);
          else mbar_arrive(go);
        }
      };
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], seq >> 1 & 1u, abort_flag))) {
        fail(ST_TIMEOUT_TMEM_FULL);
        break;
      }
      tc_fence_after();
      // the shared columns: the last of the first accumulator (the second half's), the first of the second (the first half's)
      const bool mine = buf == 0 ? part == 1 : part == 0;
      if (!mine) release();
      uint8_t* C = reinterpret_cast<uint8_t*>(p.C) + (long long)grp * p.M * p.ldc * esz;
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16) + buf * MX_ACC1 + part * cols;
      const int row0 = tm * TM + (int)half * 128 + quarter * 32, col0 = tn * q.col_tile + part * cols;
      auto read = [&]() {
        if (mine) release();
      };
      if (q.store == MX_DIRECT) mx_store_direct(p, C, taddr, row0, col0, cols, buf == 0, lane, read);
      else mx_store_staged(q, C, staging + (warp - 2) * 4096, taddr, row0, col0, cols, buf == 0, lane, read);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

template <int BT>
__global__ void __launch_bounds__(MX_GEMM_THREADS, GEMM_MIN_CTAS)
gemm_mx4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
                const __grid_constant__ CUtensorMap tmSB, MxGemmParams q) {
  extern __shared__ uint8_t smem_raw[];
  mx_gemm_cta<false, BT>(tmA, tmB, tmSA, tmSB, q, smem_raw);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MX_GEMM_THREADS, GEMM_MIN_CTAS)
gemm_mx4_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
                     const __grid_constant__ CUtensorMap tmSB, MxGemmParams q) {
  extern __shared__ uint8_t smem_raw[];
  mx_gemm_cta<true, 1>(tmA, tmB, tmSA, tmSB, q, smem_raw);
}

}  // namespace apb

using namespace apb;

extern "C" int apb_gemm_mx4_rows_takes(long long G, long long M, long long N, long long K, int values, int num_sms);
extern "C" int apb_gemm_mx4_rows(const void* A, const void* SA, const void* B, const void* SB, void* C, long long G, long long M, long long N, long long K,
                                 long long gs, long long ld, int x_type, int out_fp32, int slices, uint32_t* status, int num_sms, cudaStream_t stream);
extern "C" int apb_gemm_resident_pairs(int num_sms);
extern "C" int apb_gemm_get_reserved_sms();

// A, B: codes [G, M, kp / 2] and [G, N, kp / 2]; SA, SB: scales [G, M / 128, kp / 128, 512]; kp a multiple of 32; C [G, M, N]; all dense, 16-byte bases.
// ``form``: 0 = one CTA on 128 x 128 tiles, 1 = one CTA on 128 x 256, 2 = pairs on 256 x 256, -1 = chosen here
// (products of a few rows go to gemm_mx4_rows.cu then).
// Returns 0, or an argument / driver / launch error (nothing launched).
extern "C" int apb_gemm_mx4(const void* A, const void* SA, const void* B, const void* SB, void* C, long long G, long long M, long long N, long long kp,
                            int out_fp32, int form, uint32_t* status, int num_sms, cudaStream_t stream) {
  if (G < 0 || M < 0 || N < 0 || kp < 0 || kp % 32 || M >= 1ll << 31 || N >= 1ll << 31 || kp >= 1ll << 30 || G >= 1ll << 31) return 3;
  if (G == 0 || M == 0 || N == 0) return 0;
  for (const void* ptr : {A, SA, B, SB, (const void*)C})
    if (reinterpret_cast<uintptr_t>(ptr) & 15) return 3;
  if (kp == 0) return zero_result(C, G * M, N, N, out_fp32, stream);
  if (form < 0 && apb_gemm_mx4_rows_takes(G, M, N, kp, 0, num_sms))
    return apb_gemm_mx4_rows(A, SA, B, SB, C, G, M, N, kp, 0, 0, 2, out_fp32, 0, status, num_sms, stream);
  // Small tiles where they all run at once: 999 x 1408 x 2048 5.8 us (single 128 x 256 7.4, pairs 7.5), 128 x 4096 x 4096 7.1 (9.7, 9.7); otherwise pairs
  // (8192 x 8192 x 8192 178 us, single 128 x 256 237, 128 x 128 257; 2048 x 4096 x 4096 17.4, 18.9, 22.0), or 128 x 256 where a pair's second half
  // would have no rows.
  if (form < 0) form = G * ((M + 127) / 128) * ((N + 127) / 128) <= num_sms ? 0 : M > 128 ? 2 : 1;
  const bool pair = form == 2;
  MxGemmParams q{};
  GemmParams& p = q.p;
  p.M = (int)M;
  p.N = (int)N;
  p.C = C;
  p.ldc = N;
  p.out_fp32 = out_fp32;
  p.status = status;
  q.col_tile = form == 0 ? 128 : 256;
  const long long row_bytes = N * (out_fp32 ? 4 : 2);
  q.store = row_bytes % 32 == 0 && (reinterpret_cast<uintptr_t>(C) & 31) == 0 ? MX_DIRECT : row_bytes % 16 == 0 ? MX_STAGED : MX_SCALAR;
  q.grouped = G > 1;
  q.num_m = (int)((M + (pair ? 255 : 127)) / (pair ? 256 : 128));
  p.num_n_tiles = (int)((N + q.col_tile - 1) / q.col_tile);
  q.num_kb = (int)((kp + MX_BK - 1) / MX_BK);
  q.k_steps = (int)((kp + 63) / 64);
  const long long tiles = G * q.num_m * p.num_n_tiles;
  if (tiles >= 1ll << 30) return 3;
  q.tiles = (int)tiles;
  set_tile_order(p, q.num_m, p.num_n_tiles);
  const uint64_t words = (uint64_t)((kp + 127) / 128) * (MX_SCALE_TILE / 4);
  CUtensorMap tmA, tmB, tmSA, tmSB;
  int e = mx_map(&tmA, A, kp / 2, M, G, MX_ROW_BYTES, 128, false);
  if (!e) e = mx_map(&tmB, B, kp / 2, N, G, MX_ROW_BYTES, form == 1 ? 256 : 128, false);
  if (!e) e = mx_map(&tmSA, SA, words, (M + 127) / 128, G, MX_SC_BYTES / 4, 1, true);
  if (!e) e = mx_map(&tmSB, SB, words, (N + 127) / 128, G, MX_SC_BYTES / 4, form == 0 ? 1 : 2, true);
  if (e) return e;
  const int reserved = apb_gemm_get_reserved_sms();
  auto launch = [&](auto kern, int units, int smem) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    launch_after(kern, (unsigned)units, MX_GEMM_THREADS, smem, stream, tmA, tmB, tmSA, tmSB, q);
    return cudaGetLastError() == cudaSuccess ? 0 : 4;
  };
  if (pair) {
    const int resident = std::max(1, apb_gemm_resident_pairs(num_sms) - reserved / 2);
    return launch(gemm_mx4_pair_kernel, 2 * std::min(q.tiles, resident), MxShape<true, 1>::SMEM);
  }
  const int usable = std::max(1, num_sms - reserved);
  return form == 1 ? launch(gemm_mx4_kernel<2>, std::min(q.tiles, usable), MxShape<false, 2>::SMEM)
                   : launch(gemm_mx4_kernel<1>, std::min(q.tiles, usable), MxShape<false, 1>::SMEM);
}
