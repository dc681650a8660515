// The CTA-pair kernel behind the gated projection and its gradients (gated_forward.cu, gated_backward.cu).
//
//   GATED   out = act(x Wg) * (x Wu), optionally with P = u act'(g) and A = act(g) for the backward pass
//   SUM     out = A0 B0 + A1 B1           dx  = dG Wg^T + dU Wu^T
//   TWIN    out0 = A0 B0, out1 = A1 B1    dWg, dWu = x^T dG, x^T dU (or their transposes)
//
// The structure is that of the 256-row pair kernel of fp8_gemm.cu: two CTAs drive one M = 256 instruction
// (tcgen05.mma.cta_group::2), each loads its own 128 rows of A and half of the tile's BN columns of B, a TMA warp, an MMA
// warp and eight epilogue warps work on two accumulators in tensor memory.  What is new is where the operands come from:
//
//   GATED: the leader's half of B is BN/2 columns of Wg, the other CTA's half the SAME columns of Wu.  One instruction
//     then computes g and u of a row side by side in one accumulator, and a thread of the epilogue finds both in its
//     own tensor-memory lane: the gate costs no exchange, x is read once for both products, and g and u never leave
//     the SM.  The tensor pipe does exactly the work of one GEMM of 2F columns.
//   SUM: the K loop runs over the blocks of the first product and on over those of the second.  With few tiles the loop
//     is cut into `splits` units of work (SUM_SPLIT), whose fp32 partial sums a second kernel adds in order.
//     SUM_TALL has 512 rows a pair (256 a CTA, in two accumulators that fill tensor memory): a quarter less operand
//     traffic per product, for an epilogue that the next tile's products do not overlap.
//   TWIN: the tile index runs over both products' tiles.
//   A_MN: A is stored with its rows (M) contiguous, as x and dG are in the weights' gradients; both operands may be.
#pragma once

#include "activation.cuh"
#include "common.cuh"
#include "epilogue.cuh"
#include "gemm_tile.cuh"
#include "host.h"

namespace hb {

enum GatedMode : int { MODE_GATED = 0, MODE_GATED_TRAIN = 1, MODE_SUM = 2, MODE_TWIN = 3, MODE_SUM_SPLIT = 4, MODE_SUM_TALL = 5 };

constexpr int GG_BM = 256;      // rows of a pair's instruction
constexpr int GG_BK = 128;      // bytes of K per stage (64 rows of 16-bit values where K is not contiguous)
constexpr int GG_UMMA_K = 32;   // bytes of K per instruction
constexpr int GG_EPI_WARPS = 8;
constexpr int GG_THREADS = 64 + 32 * GG_EPI_WARPS;

template <int BN, int MODE>
struct GatedLayout {
  static constexpr bool TRAIN = MODE == MODE_GATED_TRAIN;
  static constexpr bool TALL = MODE == MODE_SUM_TALL;
  static constexpr int A_BYTES = (TALL ? 256 : 128) * GG_BK;
  static constexpr int B_BYTES = BN / 2 * GG_BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // staging of one warp: 4 KB for the output; TRAIN: 2 KB for the output and an fp32 block of 32 x 32 that P and A
  // take turns in (a second one would cost a stage of operands)
  static constexpr int WARP_EPI_BYTES = TRAIN ? 2048 + 4096 : 4096;
  static constexpr int STAGES = TALL ? 4 : (BN == 256 ? (TRAIN ? 5 : 6) : (TRAIN ? 7 : 8));
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int NUM_BARS = 2 * STAGES + 5;
  static constexpr int EPI_OFFSET = RING_BYTES;
  static constexpr int BAR_OFFSET = EPI_OFFSET + GG_EPI_WARPS * WARP_EPI_BYTES;
  static constexpr int MISC_OFFSET = BAR_OFFSET + NUM_BARS * 8;
  static constexpr int SMEM_BYTES = MISC_OFFSET + 16 + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
  static_assert(!TALL || BN == 256, "two accumulators of a tall tile fill tensor memory");
};

struct GatedMaps {
  CUtensorMap a[2], b[2];
  CUtensorMap out[3];  // GATED: out, P, A; SUM: out; TWIN: out0, out1
};

struct GatedParams {
  int M, N;        // rows and columns of out (of each out for TWIN); N counts gated columns for GATED
  int k_blocks;    // stages per product
  int splits;      // SUM_SPLIT: units the K loop is cut into
  int group_m;
  int act;
  uint32_t* status;
  const float *scale_x, *scale_w[2];  // gradients: scale_x is the factor of all results of fp16 operands
  int scale_mode;
};

// Scales 32 columns' g or u of one row.
template <int KIND>
__device__ __forceinline__ void gated_scale(uint32_t (&r)[32], const GatedParams& p, int w, int row, int col) {
  acc_to_float<KIND>(r);
  const EpiScale sc{p.scale_x, p.scale_w[w], p.scale_mode, nullptr, 0};
  scales_only_chunk(r, sc, row, p.M, col, p.N);
}

template <int ACT, bool FINE>
__device__ __forceinline__ void gate_chunk(uint32_t (&g)[32], const uint32_t (&u)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a, d;
    activate<ACT, false, FINE>(__uint_as_float(g[i]), a, d);
    g[i] = __float_as_uint(a * __uint_as_float(u[i]));
  }
}

// g -> A, u -> P, h = A u
template <int ACT>
__device__ __forceinline__ void gate_chunk_train(uint32_t (&g)[32], uint32_t (&u)[32], uint32_t (&h)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float a, d;
    const float uf = __uint_as_float(u[i]);
    activate<ACT, true, false>(__uint_as_float(g[i]), a, d);
    h[i] = __float_as_uint(a * uf);
    g[i] = __float_as_uint(a);
    u[i] = __float_as_uint(uf * d);
  }
}

template <int KIND, bool A_MN, bool B_MN, int BN, int MODE, int OUT_DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GG_THREADS, 1)
gated_pair_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
  using L = GatedLayout<BN, MODE>;
  constexpr int STAGES = L::STAGES;
  constexpr int ES = kind_bytes(KIND);
  constexpr int KROWS = GG_BK / ES;  // K rows of a stage whose K is not contiguous
  constexpr bool GATED = MODE == MODE_GATED || MODE == MODE_GATED_TRAIN;
  constexpr int TILE_N = GATED ? BN / 2 : BN;  // columns of out per tile
  constexpr bool TALL = L::TALL;
  constexpr int TILE_M = TALL ? 2 * GG_BM : GG_BM;
  static_assert(!(TALL && A_MN), "the tall tile is built for an A with K contiguous");
  constexpr int HALF_BLOCKS = BN / 2 * ES / 128;  // 128-byte column blocks of this CTA's half of an MN-major B
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFFSET);
  uint64_t* full = bars;                        // used in the leader only
  uint64_t* empty = bars + STAGES;              // one set per CTA
  uint64_t* acc_full = bars + 2 * STAGES;       // one set per CTA
  uint64_t* acc_empty = bars + 2 * STAGES + 2;  // used in the leader only (one arrival per epilogue warp of both CTAs)
  uint64_t* drain = bars + 2 * STAGES + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFFSET);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::MISC_OFFSET + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int m_tiles = (p.M + TILE_M - 1) / TILE_M;
  const int n_tiles = (p.N + TILE_N - 1) / TILE_N;
  const int one = m_tiles * n_tiles;                  // tiles of one product
  constexpr bool SUM = MODE == MODE_SUM || MODE == MODE_SUM_SPLIT || TALL;
  constexpr bool LAYERS = MODE == MODE_TWIN || MODE == MODE_SUM_SPLIT;  // one tile of out belongs to several units
  const int num_tiles = MODE == MODE_TWIN ? 2 * one : (MODE == MODE_SUM_SPLIT ? p.splits * one : one);
  const int k_all = SUM ? 2 * p.k_blocks : p.k_blocks;
  const int k_unit = MODE == MODE_SUM_SPLIT ? (k_all + p.splits - 1) / p.splits : k_all;
  const WaitCtx wctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[GATED ? rank : 0]);
    tma_prefetch_desc(&maps.out[0]);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], TALL ? GG_EPI_WARPS : 2 * GG_EPI_WARPS);  // the warps that drain it, of both CTAs
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, L::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------- TMA producer (both CTAs) --------------------------------
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        const int layer = LAYERS ? tile / one : 0;
        const TileCoord tc = tile_coord(tile - layer * one, m_tiles, n_tiles, p.group_m);
        const int k_begin = MODE == MODE_SUM_SPLIT ? layer * k_unit : 0;
        const int k_end = min(k_begin + k_unit, k_all);
        const int row0 = tc.m_blk * TILE_M + static_cast<int>(rank) * (TILE_M / 2);
        const int col0 = GATED ? tc.n_blk * TILE_N : tc.n_blk * BN + static_cast<int>(rank) * (BN / 2);
        for (int kt = k_begin; kt < k_end; ++kt, ++it) {
          const uint32_t s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1u;
          if (!mbar_wait(&empty[s], ph ^ 1u, wctx, SITE_GEMM_EMPTY)) {
            ok = false;
            break;
          }
          const int second = SUM ? (kt >= p.k_blocks ? 1 : 0) : layer;
          const int kb = SUM ? kt - second * p.k_blocks : kt;
          const CUtensorMap* ma = &maps.a[second];
          const CUtensorMap* mb = &maps.b[GATED ? static_cast<int>(rank) : second];
          uint8_t* a_dst = smem + s * L::STAGE_BYTES;
          uint8_t* b_dst = a_dst + L::A_BYTES;
          const uint32_t full_leader = map_to_cta(smem_u32(&full[s]), 0);
          if (leader) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE_BYTES);
          if constexpr (!A_MN) {
            tma_load_2d_pair(a_dst, ma, full_leader, kb * GG_BK, row0);
          } else {
            // this CTA's 128 rows = ES blocks of 128 bytes x KROWS rows of K
#pragma unroll
            for (int j = 0; j < ES; ++j) {
              tma_load_2d_pair(a_dst + j * (KROWS * 128), ma, full_leader, row0 * ES + j * 128, kb * KROWS);
            }
          }
          if constexpr (!B_MN) {
            tma_load_2d_pair(b_dst, mb, full_leader, kb * GG_BK, col0);
          } else {
#pragma unroll
            for (int j = 0; j < HALF_BLOCKS; ++j) {
              tma_load_2d_pair(b_dst + j * (KROWS * 128), mb, full_leader, col0 * ES + j * 128, kb * KROWS);
            }
          }
        }
      }
      if (!ok && leader) {
        // Abort path: the leader's `full` barriers count the bytes of both CTAs; let them land.
        const uint32_t back = it < static_cast<uint32_t>(STAGES) ? it : static_cast<uint32_t>(STAGES);
        for (uint32_t j = it - back; j < it; ++j) mbar_drain(&full[j % STAGES], (j / STAGES) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (leader CTA only) -----------------------------
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = make_idesc<KIND>(GG_BM, BN, A_MN, B_MN);
      uint32_t it = 0;
      uint32_t tile_iter = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++tile_iter) {
        // tiles take turns with the two accumulators; a tall tile fills both, each handed back on its own
        const uint32_t acc = TALL ? 0u : tile_iter & 1u;
        const uint32_t acc_ph = TALL ? tile_iter & 1u : (tile_iter >> 1) & 1u;
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, wctx, SITE_GEMM_ACC_EMPTY)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const int k_begin = MODE == MODE_SUM_SPLIT ? tile / one * k_unit : 0;
        const int k_end = min(k_begin + k_unit, k_all);
        for (int kt = k_begin; kt < k_end; ++kt, ++it) {
          const uint32_t s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1u;
          if (!mbar_wait(&full[s], ph, wctx, SITE_GEMM_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_addr = smem_u32(smem + s * L::STAGE_BYTES);
          const uint32_t b_addr = a_addr + L::A_BYTES;
          // K contiguous: 128-byte rows, 8-row atoms 1024 bytes apart.  M / N contiguous: 128-byte blocks KROWS*128
          // bytes apart, 8 K rows per atom; an instruction consumes UMMA_K/ES rows of K.
          const uint64_t b_desc = make_smem_desc(b_addr, B_MN ? KROWS * 128 : 16, 1024, SWZ_128B);
#pragma unroll
          for (int h = 0; h < (TALL ? 2 : 1); ++h) {
            if (TALL && h == 1 && kt == k_begin) {
              if (!mbar_wait(&acc_empty[1], acc_ph ^ 1u, wctx, SITE_GEMM_ACC_EMPTY)) {
                ok = false;
                break;
              }
              tc_fence_after_sync();
            }
            const uint64_t a_desc = make_smem_desc(a_addr + h * (128 * GG_BK), A_MN ? KROWS * 128 : 16, 1024, SWZ_128B);
#pragma unroll
            for (int k = 0; k < GG_BK / GG_UMMA_K; ++k) {
              const uint64_t ad = desc_advance(a_desc, k * (A_MN ? GG_UMMA_K / ES * 128 : GG_UMMA_K));
              const uint64_t bd = desc_advance(b_desc, k * (B_MN ? GG_UMMA_K / ES * 128 : GG_UMMA_K));
              umma_ss_pair<KIND>(d_tmem + h * BN, ad, bd, idesc, kt != k_begin || k != 0 ? 1u : 0u);
            }
          }
          if (!ok) break;
          const uint32_t e_local = smem_u32(&empty[s]);
          umma_commit_pair(e_local);
          umma_commit_pair(map_to_cta(e_local, 1));
        }
        if (ok) {
          const uint32_t f_local = smem_u32(&acc_full[acc]);
          umma_commit_pair(f_local);
          umma_commit_pair(map_to_cta(f_local, 1));
        }
      }
      if (!ok) {
        umma_commit_pair(smem_u32(drain));
        mbar_drain(drain, 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------- epilogue (both CTAs) -------------------------------------
    const int quarter = warp & 3;  // a warp may only touch TMEM lanes [32*(warp%4), +32)
    const int half = (warp - 2) >> 2;  // two warps share a quarter's columns (a tall tile: one for each accumulator)
    const int c_begin = TALL ? 0 : half * (TILE_N / 2), c_end = TALL ? TILE_N : (half + 1) * (TILE_N / 2);
    uint8_t* stage = smem + L::EPI_OFFSET + (warp - 2) * L::WARP_EPI_BYTES;
    uint32_t chunk_count = 0;
    uint32_t tile_iter = 0;
    const float factor = !GATED && KIND == KIND_F16 ? *p.scale_x : 1.0f;  // written by the kernel before this one
    for (int tile = pair_id; tile < num_tiles; tile += num_pairs, ++tile_iter) {
      const int layer = LAYERS ? tile / one : 0;
      const TileCoord tc = tile_coord(tile - layer * one, m_tiles, n_tiles, p.group_m);
      const uint32_t acc = TALL ? static_cast<uint32_t>(half) : tile_iter & 1u;
      const uint32_t acc_ph = TALL ? tile_iter & 1u : (tile_iter >> 1) & 1u;
      bool ok = mbar_wait(&acc_full[TALL ? 0 : acc], acc_ph, wctx, SITE_GEMM_ACC_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const int row0 = tc.m_blk * TILE_M + static_cast<int>(rank) * (TILE_M / 2) + (TALL ? half * 128 : 0) + quarter * 32;
      const uint32_t t_row = tmem_base + acc * BN + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = c_begin; c < c_end; c += 32, ++chunk_count) {
        const int col = tc.n_blk * TILE_N + c;
        const bool inside = row0 < p.M && col < p.N;
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c, r);
        if constexpr (GATED) {
          uint32_t u[32];
          tmem_ld_32x32b_x32(t_row + BN / 2 + c, u);
          tmem_wait_ld();
          gated_scale<KIND>(r, p, 0, row0 + lane, col);
          gated_scale<KIND>(u, p, 1, row0 + lane, col);
          if constexpr (MODE == MODE_GATED) {
            constexpr bool FINE = OUT_DT == HB200_DT_FP32;
            if (p.act == ACT_SILU) gate_chunk<ACT_SILU, FINE>(r, u);
            else if (p.act == ACT_GELU) gate_chunk<ACT_GELU, FINE>(r, u);
            else gate_chunk<ACT_GELU_TANH, FINE>(r, u);
            StagedStore<OUT_DT>::store(r, stage, chunk_count, lane, &maps.out[0], col, row0, inside);
          } else {
            uint32_t h[32];
            if (p.act == ACT_SILU) gate_chunk_train<ACT_SILU>(r, u, h);
            else if (p.act == ACT_GELU) gate_chunk_train<ACT_GELU>(r, u, h);
            else gate_chunk_train<ACT_GELU_TANH>(r, u, h);
            // the stores come in the order h, P, A: two lie between two uses of h's buffer, one between A's and the
            // next P's use of the other, none between P's and A's
            StagedStore<OUT_DT>::template store<2>(h, stage, 0, lane, &maps.out[0], col, row0, inside);
            StagedStore<HB200_DT_FP32>::template store<1>(u, stage + 2048, 0, lane, &maps.out[1], col, row0, inside);
            StagedStore<HB200_DT_FP32>::template store<0>(r, stage + 2048, 0, lane, &maps.out[2], col, row0, inside);
          }
        } else {
          tmem_wait_ld();
          if constexpr (KIND == KIND_F16) {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
          }
          if constexpr (MODE == MODE_SUM_SPLIT) {
            constexpr int KEEP = StagedStore<OUT_DT>::NBUF - 1;
            StagedStore<OUT_DT>::template store<KEEP, true>(r, stage, chunk_count, lane, &maps.out[0], col, row0, inside, nullptr, layer);
          } else {
            StagedStore<OUT_DT>::store(r, stage, chunk_count, lane, &maps.out[layer], col, row0, inside);
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[acc]), 0));
    }
    if (lane == 0) tma_store_wait<0>();  // all output blocks written before the CTA exits
  }

  // ------------------------------- teardown ----------------------------------------------------
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves (or frees tensor memory) while the other may still use it
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, L::TMEM_COLS);
  }
}

// ---- host side -----------------------------------------------------------------------------------

// Operand map over bytes.  K contiguous: rows of `k` elements, a box of `rows` of them.  Otherwise rows of K, `n`
// elements wide, in boxes of 128 bytes x KROWS.
inline int gated_operand_map(CUtensorMap* map, const void* base, bool mn_major, int64_t k, int64_t n, int64_t ld, int es, int rows) {
  if (!mn_major) {
    const uint64_t dims[2] = {static_cast<uint64_t>(k * es), static_cast<uint64_t>(n)};
    const uint64_t strides[1] = {static_cast<uint64_t>(ld * es)};
    const uint32_t box[2] = {GG_BK, static_cast<uint32_t>(rows)};
    return encode_tmap_u8(map, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const uint64_t dims[2] = {static_cast<uint64_t>(n * es), static_cast<uint64_t>(k)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld * es)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(GG_BK / es)};
  return encode_tmap_u8(map, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Output map of 32 x 32 boxes, swizzled like StagedStore's buffers.
inline int gated_out_map(CUtensorMap* map, void* base, int64_t m, int64_t n, int64_t ld, bool fp32) {
  const uint64_t elem = fp32 ? 4 : 2;
  const uint64_t dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld) * elem};
  const uint32_t box[2] = {32, 32};
  return encode_tmap(map, fp32 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, base, 2, dims, strides, box,
                     fp32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// The same for `layers` fp32 matrices one after another.
inline int gated_out_map_layers(CUtensorMap* map, void* base, int64_t m, int64_t n, int layers) {
  const uint64_t dims[3] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m), static_cast<uint64_t>(layers)};
  const uint64_t strides[2] = {static_cast<uint64_t>(n) * 4, static_cast<uint64_t>(m) * static_cast<uint64_t>(n) * 4};
  const uint32_t box[3] = {32, 32, 1};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Whether 128-column tiles finish earlier than 256-column ones: by the rounds of tiles over the CTA pairs.  A round of narrow
// tiles was measured at 0.83 to 0.91 of a round of wide ones (they read 3/4 of the operand bytes for half the products:
// bf16 forward 1327 x 1312 x 5784 69 us in 8 rounds against 40 us in 4), so they pay where the rounds are the same
// (222 x 480 x 400 7.2 against 8.3 us).
inline bool gated_narrow_tiles(int64_t m, int64_t columns, int products, int num_sms) {
  const int64_t pairs = num_sms / 2;
  const int64_t m_tiles = (m + GG_BM - 1) / GG_BM;
  const int64_t wide = (products * m_tiles * ((columns + 255) / 256) + pairs - 1) / pairs;
  const int64_t narrow = (products * m_tiles * ((columns + 127) / 128) + pairs - 1) / pairs;
  return narrow * 0.85 < wide * 1.0;
}

template <int KIND, bool A_MN, bool B_MN, int BN, int MODE, int OUT_DT>
int launch_gated_pair(const GatedMaps& maps, const GatedParams& p, DeviceCtx* ctx, int device, cudaStream_t stream) {
  using L = GatedLayout<BN, MODE>;
  auto kernel = gated_pair_kernel<KIND, A_MN, B_MN, BN, MODE, OUT_DT>;
  constexpr int TILE_N = MODE == MODE_GATED || MODE == MODE_GATED_TRAIN ? BN / 2 : BN;
  static std::atomic<uint64_t> smem_attr_done{0};
  HB_CUDA_CHECK(set_max_dynamic_smem_once(smem_attr_done, reinterpret_cast<const void*>(kernel), L::SMEM_BYTES, device));
  constexpr int64_t TILE_M = L::TALL ? 2 * GG_BM : GG_BM;
  const int64_t tiles = ((p.M + TILE_M - 1) / TILE_M) * ((p.N + static_cast<int64_t>(TILE_N) - 1) / TILE_N) *
                        (MODE == MODE_TWIN ? 2 : (MODE == MODE_SUM_SPLIT ? p.splits : 1));
  const int pairs = static_cast<int>(tiles < ctx->num_sms / 2 ? tiles : ctx->num_sms / 2);
  HB_CUDA_CHECK(launch_pdl(kernel, static_cast<unsigned>(2 * pairs), GG_THREADS, L::SMEM_BYTES, stream, maps, p));
  return HB200_OK;
}

}  // namespace hb
