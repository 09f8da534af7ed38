// MXFP4 products with few rows of A, sm_100a: a projection of some tokens (decoding), with the rounding of the activations in the same launch.
//
//   C[g][M, N] = A[g][M, K] * B[g][N, K]^T, M <= 32; B in 4 bits; A bf16 or fp32 values that are rounded here, or codes and scales
//
// Bound by reading B once.  B's rows take the 128 rows of the MMA and A's few rows its N, so that a stage brings in 16 KB of B and next to
// nothing of A.  A cluster of S CTAs takes a slice of K each for one tile of 128 rows of B: with as many CTAs as two to an SM, all of B's bytes that
// fit the chip's shared memory are on their way as soon as the launch has begun.  The slices' sums meet in shared memory: every CTA sends each other
// one its share of the rows, and adds up what it gets in the order of the slices - the same result every time.  With more tiles than CTAs at once a CTA has
// several, one after the other: loads, rounding and MMAs go on into the next tile while the last one's sums (two accumulators in turn) are stored.
// Measured: 1 x 14336 x 4096 from bf16 7.8 us with the weights in L2, 10 from memory (31 MB: 3.1 TB/s; a launch with its TMEM, first bytes and last stores is
// 3 us), 17 x 4096 x 14336 from codes 9.4, 32 x 4096 x 4096 7.1; 64 experts of 1408 x 2048, one row each, from memory 19 (98 MB: 80 % of the copy rate; 24.6
// with a CTA for each tile).
//   warp 0: TMA producer | warp 1: TMEM owner, scale copies, MMAs | warps 2..9: rounding of A, a stage a warp, then the epilogue
#include <algorithm>

#include "mx4.cuh"

namespace apb {

constexpr int MR_WARPS = 8, MR_THREADS = 64 + 32 * MR_WARPS, MR_MAX_STAGES = 8;
constexpr int MR_SMEM = 112 * 1024;  // two CTAs to an SM

struct MxRowsParams {
  const void* x;  // values of A (rounded here), or null
  void* C;
  int M, N, K, tiles, n_tiles, num_kb, k_steps, slices, stages, vec, out_fp32;
  FastDiv div_tiles, div_blocks;  // by the tiles of a matrix, by the k-blocks of a tile
  long long gs, ld;
  uint32_t* status;
};

// NT: columns of the MMA (rows of A, padded)
template <int NT>
struct MxRowsShape {
  static constexpr int STAGE = MX_OP_BYTES + 2 * MX_SC_BYTES + NT * MX_ROW_BYTES;
  static constexpr int PART = NT * 128 * 4;  // sums of all slices for a CTA's share of the rows
  static constexpr int STAGES = std::min(MR_MAX_STAGES, (MR_SMEM - 1024 - 256 - PART) / STAGE);
  static constexpr int SMEM = 1024 + STAGES * STAGE + PART + 256;
  static constexpr uint32_t COLS = NT <= 16 ? 64 : 128;  // TMEM: sums of two tiles, 16 columns of scales
};

// Four rows of a stage of A, one warp: a lane has 8 values of each, four lanes a block.
template <typename T>
struct MxRowsUnit {
  static constexpr int W = 8 * (int)sizeof(T) / 4;
  uint32_t u[4][W];
  __device__ __forceinline__ void load(const MxRowsParams& p, const T* x, int r0, int k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int c = 0; c < W; ++c) u[i][c] = 0;
      if (r0 + i >= p.M) continue;
      const T* src = x + (r0 + i) * p.ld + k;
      if (p.vec) {
        if (k < p.K) {
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(src) + c);
            u[i][c] = v.x, u[i][c + 1] = v.y, u[i][c + 2] = v.z, u[i][c + 3] = v.w;
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (k + c < p.K) mx_put(u[i], c, src[c]);
      }
    }
  }
  __device__ __forceinline__ void round(const MxRowsParams& p, int r0, uint8_t* op, uint8_t* sc, int lane) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i;
      if (r >= p.M) break;
      uint32_t m = 0;
#pragma unroll
      for (int c = 0; c < W; ++c) m = mx_word_max<T>(m, u[i][c]);
      uint32_t amax = mx_word_max_bits<T>(m);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const uint32_t code = mx_scale_code(amax);
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = mx_word_value<T>(u[i], c);
      *reinterpret_cast<uint32_t*>(op + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = mx_encode_block(v, code);
      if ((lane & 3) == 0) sc[(lane >> 4) * MX_SCALE_TILE + mx_scale_at(r, lane >> 2 & 3)] = (uint8_t)code;
    }
  }
};

template <int NT, typename T>  // T: type of A's values; void: codes
__global__ void __launch_bounds__(MR_THREADS, 2)
gemm_mx4_rows_kernel(const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ MxRowsParams p) {
  using S = MxRowsShape<NT>;
  constexpr bool VALUES = !std::is_same<T, void>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sB = smem;                                       // [stages] 16 KB of B, then
  uint8_t* sA = sB + p.stages * MX_OP_BYTES;                // [stages] NT rows of A, then
  uint8_t* sSc = sA + p.stages * NT * MX_ROW_BYTES;         // [stages] scales of B, of A
  float* part = reinterpret_cast<float*>(sSc + p.stages * 2 * MX_SC_BYTES);  // [slices][NT][rows of this CTA's share]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(part) + S::PART);
  uint64_t *full = bars, *empty = bars + MR_MAX_STAGES, *acc_full = bars + 2 * MR_MAX_STAGES, *acc_free = acc_full + 2, *parts_in = acc_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(parts_in + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert((2 * MR_MAX_STAGES + 6) * 8 <= 256, "barrier block");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.slices > 1 ? (int)cluster_ctarank() : 0, first_tile = blockIdx.x / p.slices, tile_step = gridDim.x / p.slices;
  const int kb0 = p.num_kb * rank / p.slices, kb1 = p.num_kb * (rank + 1) / p.slices;
  auto place = [&](int tile, int& grp, int& n0) {
    grp = p.div_tiles.div(tile);
    n0 = (tile - grp * p.n_tiles) * 128;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], VALUES ? 1 + (p.M + 3) / 4 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_free[b], MR_WARPS);
    }
    mbar_init(parts_in, p.slices * MR_WARPS);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSB);
    if (!VALUES) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmSA);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (p.slices > 1) {
    cluster_arrive();  // every CTA's barriers are there before a peer's sums arrive
    cluster_wait();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_previous();

  auto fail = [&](uint32_t code) {
    atomicCAS(p.status, 0u, code);
    *abort_flag = 1;
  };
  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
        int grp, n0;
        place(t, grp, n0);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_EMPTY);
            break;
          }
          mbar_expect_tx(&full[stage], MX_OP_BYTES + MX_SC_BYTES + (VALUES ? 0 : NT * MX_ROW_BYTES + MX_SC_BYTES));
          uint8_t* sc = sSc + stage * 2 * MX_SC_BYTES;
          tma_load_3d(sB + stage * MX_OP_BYTES, &tmB, &full[stage], kb * MX_ROW_BYTES, n0, grp);
          tma_load_3d(sc, &tmSB, &full[stage], kb * (MX_SC_BYTES / 4), n0 / 128, grp);
          if (!VALUES) {
            tma_load_3d(sA + stage * NT * MX_ROW_BYTES, &tmA, &full[stage], kb * MX_ROW_BYTES, 0, grp);
            tma_load_3d(sc + MX_SC_BYTES, &tmSA, &full[stage], kb * (MX_SC_BYTES / 4), 0, grp);
          }
          if (++stage == p.stages) stage = 0, phase ^= 1;
        }
      }
      let_next_in();
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc[2] = {make_idesc_mx4(128, NT, 0), make_idesc_mx4(128, NT, 2)};
      const uint64_t b_desc = make_smem_desc(smem_u32(sB), 16, 1024), a_desc = make_smem_desc(smem_u32(sA), 16, 1024);
      const uint64_t sc_desc = make_scale_desc(smem_u32(sSc));
      const uint32_t sb_tmem = tmem + 2 * NT, sa_tmem = sb_tmem + 4 * MX_STAGE_TILES;
      int stage = 0;
      uint32_t phase = 0, seq = 0;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += tile_step, ++seq) {
        const uint32_t buf = seq & 1u, d_tmem = tmem + buf * NT;
        if (seq > 1 && !mbar_wait(&acc_free[buf], ((seq >> 1) - 1) & 1u, abort_flag)) {
          fail(ST_TIMEOUT_TMEM_EMPTY);
          break;
        }
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            ok = false;
            fail(ST_TIMEOUT_FULL);
            break;
          }
          tc_fence_after();
          const int steps = min(MX_BK / 64, p.k_steps - kb * (MX_BK / 64));
#pragma unroll
          for (int a = 0; a < MX_STAGE_TILES; ++a) {
            tmem_copy_scales(sb_tmem + 4 * a, sc_desc + desc_offset(stage * 2 * MX_SC_BYTES + a * MX_SCALE_TILE));
            tmem_copy_scales(sa_tmem + 4 * a, sc_desc + desc_offset(stage * 2 * MX_SC_BYTES + MX_SC_BYTES + a * MX_SCALE_TILE));
          }
#pragma unroll
          for (int s = 0; s < MX_BK / 64; ++s) {
            if (s >= steps) break;
            umma_mx4(d_tmem, b_desc + desc_offset(stage * MX_OP_BYTES + 32 * s), a_desc + desc_offset(stage * NT * MX_ROW_BYTES + 32 * s), idesc[s & 1],
                     sb_tmem + 4 * (s / 2), sa_tmem + 4 * (s / 2), kb > kb0 || s > 0 ? 1u : 0u);
          }
          umma_commit(&empty[stage]);
          if (++stage == p.stages) stage = 0, phase ^= 1;
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
    }
  } else {
    // Epilogue of this CTA's ``seq``-th tile: a warp has 32 rows of B (a TMEM lane quarter) and half of A's rows.
    const int w = warp - 2, quarter = warp & 3, half = w >> 2, row = quarter * 32 + lane;
    constexpr int COLS = NT / 2;
    auto columns = [&](uint32_t buf, auto store) {  // store(row of A, sum)
#pragma unroll
      for (int c0 = 0; c0 < COLS; c0 += 8) {
        if (half * COLS + c0 >= p.M) break;
        uint32_t r[8];
        tmem_ld_32x8(tmem + (uint32_t(quarter * 32) << 16) + buf * NT + half * COLS + c0, r);
        tmem_ld_wait_for8(r);
#pragma unroll
        for (int c = 0; c < 8; ++c) store(half * COLS + c0 + c, r[c]);
      }
    };
    auto put = [&](long long at, float v) {
      if (p.out_fp32) reinterpret_cast<float*>(p.C)[at] = v;
      else reinterpret_cast<__nv_bfloat16*>(p.C)[at] = __float2bfloat16(v);
    };
    auto epilogue = [&](int seq) {
      const uint32_t buf = seq & 1;
      int grp, n0;
      place(first_tile + seq * tile_step, grp, n0);
      const bool done = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], seq >> 1 & 1, abort_flag));
      if (!done) fail(ST_TIMEOUT_TMEM_FULL);
      tc_fence_after();
      if (p.slices == 1) {
        if (!done) return false;
        const long long at = (long long)grp * p.M * p.N + n0 + row;
        const bool in = n0 + row < p.N;
        columns(buf, [&](int m, uint32_t v) {
          if (in && m < p.M) put(at + (long long)m * p.N, __uint_as_float(v));
        });
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_free[buf]);
        return true;
      }
      const int share = 128 / p.slices;  // rows of B that a CTA of the cluster adds up
      if (done) {
        const uint32_t dst = map_to_cta(part + (rank * NT) * share + row % share, row / share);
        columns(buf, [&](int m, uint32_t v) { st_cluster_u32(dst + m * share * 4, v); });
      }
      __syncwarp();
      if (lane == 0)
        for (int s = 0; s < p.slices; ++s) mbar_arrive_cluster(map_to_cta(parts_in, s));
      const bool got = __all_sync(0xffffffffu, mbar_wait_cluster(parts_in, 0, abort_flag));
      if (!got) fail(ST_TIMEOUT_TMEM_FULL);
      if (!got || !done) return false;
      const int first = n0 + rank * share;
      for (int i = threadIdx.x - 64; i < p.M * share; i += 32 * MR_WARPS) {
        const int m = i / share, r = i - m * share;
        float v = 0.f;
        for (int s = 0; s < p.slices; ++s) v += part[(s * NT + m) * share + r];
        if (first + r < p.N) put(((long long)grp * p.M + m) * p.N + first + r, v);
      }
      return true;
    };
    const int my_tiles = (p.tiles - first_tile + tile_step - 1) / tile_step, per_tile = kb1 - kb0;
    int read_out = 0;  // tiles
    bool ok = true;
    if constexpr (VALUES) {
      // Units of four rows of a stage.  Every unit of a ring slot belongs to one warp, in every round of the ring: a warp that skipped a round could
      // not tell from a barrier's parity whether the slot is free or two rounds behind.
      const int groups = (p.M + 3) / 4, units = p.stages * groups, count = my_tiles * per_tile;
      struct At {
        int round, unit;
      };
      auto stage_of = [&](const At& a) { return a.unit / groups; };
      auto block_of = [&](const At& a) { return a.round * p.stages + stage_of(a); };  // k-block of this CTA
      auto after = [&](At a) {
        a.unit += MR_WARPS;
        if (a.unit >= units) a = {a.round + 1, w};
        return a;
      };
      auto load = [&](MxRowsUnit<T>& u, const At& a) {
        const int b = block_of(a);
        if (b >= count) return;
        const int seq = p.slices > 1 ? 0 : (int)p.div_blocks.div(b);
        int grp, n0;
        place(first_tile + seq * tile_step, grp, n0);
        u.load(p, reinterpret_cast<const T*>(p.x) + grp * p.gs, a.unit % groups * 4, (kb0 + b - seq * per_tile) * MX_BK + lane * 8);
      };
      MxRowsUnit<T> next;
      At at{0, w};
      const int rounds = w < units ? (count + p.stages - 1) / p.stages : 0;
      if (rounds > 0) load(next, at);
      while (at.round < rounds) {
        const MxRowsUnit<T> unit = next;
        const At then = after(at);
        if (then.round < rounds) load(next, then);
        const int b = block_of(at);
        if (b < count) {
          // A tile is read out a ring behind its last block.  What this slot waits for is an MMA of the next tile then, whose accumulator was free
          // before: no warp waits for a tile that another one has still to read out.
          while (ok && (read_out + 1) * per_tile + p.stages <= b) ok = epilogue(read_out++);
          const int stage = stage_of(at);
          if (!ok || !__all_sync(0xffffffffu, mbar_wait(&empty[stage], (at.round & 1) ^ 1, abort_flag))) {
            ok = false;
            fail(ST_TIMEOUT_EMPTY);
            break;
          }
          unit.round(p, at.unit % groups * 4, sA + stage * NT * MX_ROW_BYTES, sSc + stage * 2 * MX_SC_BYTES + MX_SC_BYTES, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        }
        at = then;
      }
    }
    while (read_out < my_tiles && (ok || p.slices > 1)) ok = epilogue(read_out++) && ok;  // (a cluster waits for all its CTAs' parts)
  }
  tc_fence_before();
  __syncthreads();
  if (p.slices > 1 && *abort_flag) {  // (one that gave up waiting: the others, which may still write to it, leave or come here first)
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::COLS);
  }
}

}  // namespace apb

using namespace apb;

extern "C" int apb_gemm_get_reserved_sms();

// CTAs that are there at once: two to an SM.
static long long mx_rows_resident(int num_sms) { return 2ll * std::max(1, num_sms - apb_gemm_get_reserved_sms()); }

// Slices of K for a product of ``tiles`` tiles of 128 rows of B: as many as are resident at once, each with a stage at least.
static int mx_rows_slices(long long tiles, int num_kb, long long resident) {
  int s = 1;
  while (s < 4 && tiles * 2 * s <= resident && 4 * s <= num_kb) s *= 2;
  return s;
}

// Whether a product with M rows of A is this file's.  us, with weights from memory:
//   codes                  this kernel / the persistent ones of gemm_mx4.cu: 64 experts of 1408 x 2048 2 rows 19.3 / 20.9, 16 rows 20.0 / 21.6, 32 rows 20.4 / 22.1;
//                          16 of 4096 x 4096 26.5 / 29.0 (8 rows); 128 of 768 x 2048 21.0 / 22.5; 16 x 14336 x 4096 10.9, in L2 8.6 / 10.1; 32 x 40000 x 4096
//                          21.7 / 25.7; 32 x 128256 x 4096 49.6 / 56.7; in L2 17 x 4096 x 14336 9.4 / 15.3, 32 x 4096 x 4096 7.1 / 9.6
//   values, rounded here   this kernel / a launch that rounds A and the codes.  Every CTA rounds all rows of its slices of A, so more rows, and more blocks of K
//                          a CTA, are better rounded once.  Up to 4 rows (in L2, from memory): 1 x 14336 x 4096 7.3 / 9.3, 9.5 / 10.9, 4 rows 8.4 / 9.9, 9.9 / 11.0;
//                          4 x 4096 x 14336 9.3 / 9.7, 10.2 / 11.6; 64 experts of 1408 x 2048, 4 rows, 15.1 / 16.6, 18.1 / 21.2.  8 rows with 4 blocks a CTA or
//                          fewer: 4096 x 4096 6.2 / 6.6, 6.8 / 7.6; 14336 x 2048 7.5 / 7.5, 8.5 / 9.6; 8 experts of 4096 x 1024 5.8 / 5.9, 7.3 / 7.8.  With more:
//                          4096 x 6144 8.3 / 7.1, 9.0 / 8.4; 14336 x 4096 10.6 / 8.8, 11.8 / 11.5; 8 experts of 4096 x 2048 9.0 / 7.2, 10.9 / 10.9.
//                          (9 of 140 pairs, 5 and 8 rows of 8 to 256 tiles of 2 to 56 blocks, lie on the wrong side, by 5 % at most.)
extern "C" int apb_gemm_mx4_rows_takes(long long G, long long M, long long N, long long K, int values, int num_sms) {
  if (!values || M <= 4) return M <= 32;
  const long long tiles = G * ((N + 127) / 128), resident = mx_rows_resident(num_sms), blocks = (K + MX_BK - 1) / MX_BK;
  return M <= 8 && tiles <= resident && blocks <= 4 * mx_rows_slices(tiles, (int)blocks, resident);
}

// A: values [G, M, K] with unit stride along K (x_type 0: fp32, 1: bf16; up to 16 rows, more are rounded before), or codes (x_type 2) with scales SA;
// B: codes [G, N, kp / 2], scales SB; C [G, M, N] dense.  ``slices``: 1, 2 or 4, 0: chosen here.
extern "C" int apb_gemm_mx4_rows(const void* A, const void* SA, const void* B, const void* SB, void* C, long long G, long long M, long long N, long long K,
                                 long long gs, long long ld, int x_type, int out_fp32, int slices, uint32_t* status, int num_sms, cudaStream_t stream) {
  if (G < 0 || M < 0 || N < 0 || K < 0 || M > (x_type == 2 ? 32 : 16) || N >= 1ll << 31 || K >= 1ll << 30 || G >= 1ll << 31) return 3;
  if (G == 0 || M == 0 || N == 0) return 0;
  if ((reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(SB) | reinterpret_cast<uintptr_t>(C)) & 15) return 3;
  if (x_type == 2 && ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(SA)) & 15)) return 3;
  if (K == 0) return zero_result(C, G * M, N, N, out_fp32, stream);
  const long long kp = (K + 31) / 32 * 32, n_tiles = (N + 127) / 128, tiles = G * n_tiles;
  MxRowsParams p{};
  p.x = x_type == 2 ? nullptr : A;
  p.C = C;
  p.M = (int)M, p.N = (int)N, p.K = (int)K, p.tiles = (int)tiles, p.n_tiles = (int)n_tiles;
  p.num_kb = (int)((kp + MX_BK - 1) / MX_BK);
  p.k_steps = (int)((kp + 63) / 64);
  const long long resident = mx_rows_resident(num_sms);
  p.slices = slices > 0 ? slices : mx_rows_slices(tiles, p.num_kb, resident);
  p.div_tiles = FastDiv((uint32_t)n_tiles);
  p.div_blocks = FastDiv((uint32_t)p.num_kb);
  if ((p.slices & (p.slices - 1)) || p.slices > 4 || p.slices > p.num_kb || tiles * p.slices >= 1ll << 31) return 3;
  p.out_fp32 = out_fp32;
  p.gs = gs, p.ld = ld;
  p.status = status;
  const int esz = x_type == 1 ? 2 : 4;
  p.vec = x_type != 2 && ld * esz % 16 == 0 && gs * esz % 16 == 0 && K % 8 == 0 && (reinterpret_cast<uintptr_t>(A) & 15) == 0;
  const uint64_t words = (uint64_t)((kp + 127) / 128) * (MX_SCALE_TILE / 4);
  const int nt = M <= 16 ? 16 : 32;
  CUtensorMap tmB, tmSB, tmA{}, tmSA{};
  int e = mx_map(&tmB, B, kp / 2, N, G, MX_ROW_BYTES, 128, false);
  if (!e) e = mx_map(&tmSB, SB, words, n_tiles, G, MX_SC_BYTES / 4, 1, true);
  if (!e && x_type == 2) e = mx_map(&tmA, A, kp / 2, M, G, MX_ROW_BYTES, nt, false);
  if (!e && x_type == 2) e = mx_map(&tmSA, SA, words, 1, G, MX_SC_BYTES / 4, 1, true);
  if (e) return e;
  auto launch = [&](auto kern, int smem, int stages) {
    p.stages = stages;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaLaunchAttribute attr[2];
    int n = 0;
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = p.slices, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
    if (!apb_gemm_makes_room()) attr[n++] = overlap_attribute();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.slices > 1 ? tiles * p.slices : std::min(tiles, resident)));
    cfg.blockDim = dim3(MR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, tmB, tmSB, tmA, tmSA, p) == cudaSuccess ? 0 : 4;
  };
#define APB_MX_ROWS(NT, T) return launch(gemm_mx4_rows_kernel<NT, T>, MxRowsShape<NT>::SMEM, MxRowsShape<NT>::STAGES)
  if (x_type == 2) {
    if (nt == 16) APB_MX_ROWS(16, void);
    APB_MX_ROWS(32, void);
  }
  if (x_type == 1) APB_MX_ROWS(16, __nv_bfloat16);
  APB_MX_ROWS(16, float);
#undef APB_MX_ROWS
}
