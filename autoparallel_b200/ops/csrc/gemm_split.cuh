// Body of the split GEMM's CTA (gemm_split.cu says what it is for): one 128 x BN_T tile per cluster, the contraction split over the cluster's CTAs.
// Shared by the plain products and by those of the gated feed-forward block (gemm_gated.cu).
#pragma once
#include "gemm_core.cuh"

namespace apb {

constexpr int SPLIT_MAX = 8;  // portable cluster size
constexpr int SPLIT_STAGE_TOTAL = 196608;  // 8 x 24 KB, 6 x 32 KB or 4 x 48 KB: deep enough for one CTA to hide the load latency
constexpr int SPLIT_THREADS = GEMM_PLAIN_THREADS;
constexpr int SPLIT_SMEM_BYTES = SPLIT_STAGE_TOTAL + 1024 + 256;

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

namespace split {

template <bool A_MN, bool B_MN, int BN_T, bool GROUPED, typename Ext = NoExt>
__device__ __forceinline__ void gemm_cta(const CUtensorMap& tmA, const CUtensorMap& tmB, const GemmParams& p, const Ext& ext = Ext{}) {
  constexpr int EXT = Ext::KIND;
  static_assert(EXT == EXT_NONE || !GROUPED, "extended products: one problem");
  static_assert(EXT != EXT_GATED || (!A_MN && !B_MN), "both projections: K-major operands");
  constexpr int B_BYTES = BN_T * BK * 2;
  constexpr int ST = SPLIT_STAGE_TOTAL / (A_STAGE_BYTES + B_BYTES);
  constexpr int HALVES = BN_T >= 128 ? EPI_WARPS / 4 : 1, COLS = BN_T / HALVES;  // warps per lane quarter, and their columns: blocks of 64
  constexpr int LD = BN_T + 4;  // floats per row of the fp32 tile: rows start 16 bytes apart modulo the banks
  static_assert(BM * LD * 4 <= SPLIT_STAGE_TOTAL, "the fp32 tile reuses the stages");
  static_assert((2 * ST + 1) * 8 + 8 <= 256, "barrier block");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * A_STAGE_BYTES;
  float* tile = reinterpret_cast<float*>(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SPLIT_STAGE_TOTAL);
  uint64_t* empty = full + ST;
  uint64_t* tmem_full = empty + ST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int S = (int)cluster_size(), slice = (int)cluster_ctarank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_group = p.num_m_tiles * p.num_n_tiles;
  const int t = blockIdx.x / S;
  const int grp = GROUPED ? t / per_group : 0;
  int tm, tn;
  tile_coords(GROUPED ? t - grp * per_group : t, p.num_m_tiles, p.num_n_tiles, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN_T;
  const int rows = min(BM, p.M - m0);  // of the tile that are inside the matrix
  const bool solo = S == 1 && p.vec_store && EXT != EXT_GATED && EXT != EXT_GRAD;
  const int num_kb = (p.K + BK - 1) / BK;
  const int kb0 = (int)((long long)num_kb * slice / S), kb1 = (int)((long long)num_kb * (slice + 1) / S);  // S <= num_kb: never empty

  // The producer goes on as soon as it has set up the barriers; the others wait for them and for the TMEM columns, whose allocation
  // (half a microsecond) the first loads hide.
  uint32_t tmem_base = 0;
  if (warp == 0) {
    if (elect_one()) {
      for (int s = 0; s < ST; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(tmem_full, 1);
      *abort_flag = 0;
      mbar_fence_init();
    }
    __syncwarp();
    named_arrive(1, SPLIT_THREADS);
    wait_previous();
  } else {
    if (warp == 1) {
      tmem_alloc(tmem_slot, BN_T);
      tmem_relinquish();
    } else if (warp == 2 && lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
    }
    tc_fence_before();
    named_sync(1, SPLIT_THREADS);
    tc_fence_after();
    tmem_base = *tmem_slot;
    wait_previous();
  }
  auto fail = [&](uint32_t code) {
    atomicCAS(p.status, 0u, code);
    *abort_flag = 1;
  };

  // One elected thread per role, the stages unrolled, so that the barriers, the shared-memory addresses and the descriptors of a
  // stage are constants added to a base: issue is what bounded a k-block before (293 ns at any tile width, with lane 0 chosen by a
  // comparison and descriptors built from scratch; now 115 at 64 columns, 148 at 128, 277 - the tensor core's time - at 256).
  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      uint32_t phase = 1;
      for (int kb = kb0; kb < kb1 && ok; kb += ST, phase ^= 1) {
#pragma unroll
        for (int stage = 0; stage < ST; ++stage) {
          if (kb + stage >= kb1) break;
          if (!mbar_wait(&empty[stage], phase, abort_flag)) {
            fail(ST_TIMEOUT_EMPTY);
            ok = false;
            break;
          }
          auto load = [&](uint8_t* dst, const CUtensorMap* m, int x, int y) {
            if constexpr (EXT == EXT_DUAL) {  // the second half of the blocks belongs to the second pair of operands
              if (kb + stage >= num_kb / 2) {
                m = m == &tmA ? &ext.tmA2 : &ext.tmB2;
                (A_MN && m == &ext.tmA2) || (B_MN && m == &ext.tmB2) ? y -= num_kb / 2 * BK : x -= num_kb / 2 * BK;
              }
            }
            if (GROUPED) tma_load_3d(dst, m, &full[stage], x, y, grp);
            else tma_load_2d(dst, m, &full[stage], x, y);
          };
          mbar_expect_tx(&full[stage], A_STAGE_BYTES + B_BYTES);
          uint8_t* a_dst = sA + stage * A_STAGE_BYTES;
          uint8_t* b_dst = sB + stage * B_BYTES;
          const int k0 = (kb + stage) * BK;
          if (!A_MN) {
            load(a_dst, &tmA, k0, m0);
          } else {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) load(a_dst + c * CHUNK_BYTES, &tmA, m0 + c * 64, k0);
          }
          if constexpr (EXT == EXT_GATED) {
            load(b_dst, &tmB, k0, n0 / 2);
            load(b_dst + B_BYTES / 2, &ext.tmB2, k0, n0 / 2);
          } else if (!B_MN) {
            load(b_dst, &tmB, k0, n0);
          } else {
#pragma unroll
            for (int c = 0; c < BN_T / 64; ++c) load(b_dst + c * CHUNK_BYTES, &tmB, n0 + c * 64, k0);
          }
        }
      }
      let_next_in();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_bf16(BM, BN_T, A_MN ? 1u : 0u, B_MN ? 1u : 0u);
      const uint64_t a_desc = make_smem_desc(smem_u32(sA), A_MN ? CHUNK_BYTES : 16, 1024);
      const uint64_t b_desc = make_smem_desc(smem_u32(sB), B_MN ? CHUNK_BYTES : 16, 1024);
      bool ok = true;
      uint32_t phase = 0, accumulate = 0;
      for (int kb = kb0; kb < kb1 && ok; kb += ST, phase ^= 1) {
#pragma unroll
        for (int stage = 0; stage < ST; ++stage) {
          if (kb + stage >= kb1) break;
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            fail(ST_TIMEOUT_FULL);
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            umma_f16(tmem_base, a_desc + desc_offset(stage * A_STAGE_BYTES + k * (A_MN ? UMMA_K * 128 : UMMA_K * 2)),
                     b_desc + desc_offset(stage * B_BYTES + k * (B_MN ? UMMA_K * 128 : UMMA_K * 2)), idesc, k > 0 ? 1u : accumulate);
            accumulate = 1;
          }
          umma_commit(&empty[stage]);
        }
      }
      if (ok) umma_commit(tmem_full);
    }
    __syncwarp();
  } else if (warp < 2 + 4 * HALVES) {
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    const int col0 = ((warp - 2) >> 2) * COLS;  // first of its columns
    // (the TMEM loads are warp-wide: the warp goes on together or not at all)
    if (!__all_sync(0xffffffffu, mbar_wait(tmem_full, 0, abort_flag))) {
      fail(ST_TIMEOUT_TMEM_FULL);
    } else if (solo) {
      tc_fence_after();
      uint8_t* stg = smem + (warp - 2) * STORE_BYTES;
      const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + col0;
      const long long c_off = GROUPED ? (long long)grp * p.M * p.ldc : 0;
      auto nothing = []() {};
      if (p.out_fp32) store_tile<true>(reinterpret_cast<float*>(p.C) + c_off, p.ldc, stg, taddr, m0 + q * 32, n0 + col0, COLS, p.M, p.N, lane, nothing, ext);
      else store_tile<false>(reinterpret_cast<__nv_bfloat16*>(p.C) + c_off, p.ldc, stg, taddr, m0 + q * 32, n0 + col0, COLS, p.M, p.N, lane, nothing, ext);
    } else if (q * 32 < rows) {
      tc_fence_after();
      float* row = tile + (q * 32 + lane) * LD + col0;
#pragma unroll (COLS > 64 ? 2 : 4)  // (the registers of four loads are more than a communication kernel's CTA leaves)
      for (int c = 0; c < COLS / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + (uint32_t(q * 32) << 16) + col0 + c * 32, r);
        tmem_ld_wait_for(r);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          reinterpret_cast<uint4*>(row + c * 32)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
      }
    }
  }
  if (solo) {  // nothing to add up: the warps have stored the tile from TMEM
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, BN_T);
    }
    return;
  }
  tc_fence_before();
  __syncwarp();
  cluster_arrive();  // (also orders the threads of a cluster of one CTA)
  cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, BN_T);
  }

  // The sum: four columns per thread and row, the rows of a thread a whole stride apart, two at a time so that their loads are under way
  // together (the other CTAs' shared memory gives 16 bytes a cycle and SM, with a round trip of hundreds of cycles).  The loops stay small on
  // purpose: eight rows at a time, unrolled, were slower in every product (64 x 1408 x 2048 6.9 us against 5.8): the code is fetched once
  // per launch.  128 x 128 tiles in two slices: sum and store 2.8 -> 1.6 us, in one 2.8 + 0.8 -> 1.2 (TMEM to C).
  if constexpr (EXT == EXT_GATED || EXT == EXT_GRAD) {
    // (eight threads have 32 columns of one row, which share a scale of 8-bit codes: they stay together)
    constexpr int WIDTH = EXT == EXT_GATED ? BN_T / 2 : BN_T, VPR = WIDTH / 4, RSTEP = SPLIT_THREADS / VPR;
    static_assert(RSTEP * VPR == SPLIT_THREADS && VPR % 8 == 0, "whole rows");
    const int c = (threadIdx.x % VPR) * 4, H = EXT == EXT_GATED ? p.N / 2 : p.N, col = (EXT == EXT_GATED ? n0 / 2 : n0) + c;
    const uint32_t src0 = smem_u32(tile) + c * 4;
    const int first = slice * RSTEP + threadIdx.x / VPR, step = S * RSTEP;
    auto add = [](float (&a)[4], const float4& x) { a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w; };
    [[maybe_unused]] AbFour<ext_bits<Ext>()> next;  // (backward: a and b of the row after the one in work are under way)
    if constexpr (EXT == EXT_GRAD) {
      if (first < rows && col < H) next.load(ext.grad, m0 + first, col, H);
    }
#pragma unroll 1
    for (int r = *abort_flag == 0 ? first : rows; r < rows; r += step) {
      const uint32_t src = src0 + r * (LD * 4);
      float v[4] = {}, w[4] = {};
      [[maybe_unused]] const AbFour<ext_bits<Ext>()> ab = next;
      if constexpr (EXT == EXT_GRAD) {
        if (r + step < rows && col < H) next.load(ext.grad, m0 + r + step, col, H);
      }
#pragma unroll 2
      for (int s = 0; s < S; ++s) {
        const uint32_t from = map_to_cta(src, (uint32_t)s);
        const float4 x = ld_cluster_f4(from);
        if constexpr (EXT == EXT_GATED) add(w, ld_cluster_f4(from + WIDTH * 4));
        add(v, x);
      }
      if constexpr (EXT == EXT_GATED) {
        gated_four<Ext::BITS>(ext.out, m0 + r, col, H, v, w);
      } else {
        if (col < H) gated_grad_four<Ext::BITS>(ext.grad, ab, m0 + r, col, H, v);
      }
    }
  } else if (*abort_flag == 0) {
    constexpr int VPR = BN_T / 4, RSTEP = SPLIT_THREADS / VPR;  // threads per row, rows per pass of the CTA
    static_assert(RSTEP * VPR == SPLIT_THREADS, "whole rows");
    const int c = (threadIdx.x % VPR) * 4, col = n0 + c, step = S * RSTEP;
    const bool whole = (p.ldc & 3) == 0 && col + 4 <= p.N;
    const int esz = p.out_fp32 ? 4 : 2;
    const uint32_t src0 = smem_u32(tile) + c * 4;
    uint8_t* dst0 = reinterpret_cast<uint8_t*>(p.C) + ((GROUPED ? (long long)grp * p.M * p.ldc : 0) + (long long)m0 * p.ldc + col) * esz;
    const long long ld_bytes = p.ldc * esz;
    auto add = [](float4& a, const float4& x) { a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w; };
    auto store = [&](int r, const float4& v) {
      uint8_t* dst = dst0 + r * ld_bytes + row_jump(ext, m0 + r);
      if (whole) {
        if (p.out_fp32) *reinterpret_cast<float4*>(dst) = v;
        else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      } else {
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (col + i >= p.N) break;
          if (p.out_fp32) reinterpret_cast<float*>(dst)[i] = f[i];
          else reinterpret_cast<__nv_bfloat16*>(dst)[i] = __float2bfloat16(f[i]);
        }
      }
    };
#pragma unroll 1
    for (int r = slice * RSTEP + threadIdx.x / VPR; r < rows && col < p.N; r += 2 * step) {
      const uint32_t src = src0 + r * (LD * 4);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (r + step < rows) {
#pragma unroll 2
        for (int s = 0; s < S; ++s) {
          const uint32_t from = map_to_cta(src, (uint32_t)s);
          const float4 x = ld_cluster_f4(from), y = ld_cluster_f4(from + step * (LD * 4));
          add(a, x);
          add(b, y);
        }
        store(r + step, b);
      } else {
#pragma unroll 4
        for (int s = 0; s < S; ++s) add(a, ld_cluster_f4(map_to_cta(src, (uint32_t)s)));
      }
      store(r, a);
    }
  }
  __syncwarp();
  cluster_arrive_relaxed();  // no CTA leaves while another may still read its tile
  cluster_wait();
}

}  // namespace split
}  // namespace apb
