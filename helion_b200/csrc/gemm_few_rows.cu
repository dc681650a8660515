// Products of few rows (M <= 128) with one or two column-major weights: int8_gemm for a handful of tokens, and the
// gated projection act(x Wg) * (x Wu) for them (e4m3, int8, fp16 or bf16 operands).  int8_gemm also has more rows of x
// computed here, in blocks of 256, where the columns are so few that tiles would leave most SMs idle and K is split.
//
// Such a call is bound by reading the weights once.  As in fp8_gemm_skinny.cu the operands are swapped: 128 rows of the
// tensor-core tile are columns of the weight (K contiguous), the rows of x are its N dimension.  Two things differ:
//
//   - the columns are shared out evenly: a CTA takes R = ceil(columns / SMs) of them, any number up to 128, so every
//     SM streams the same bytes (14336 columns on 148 SMs are 97 each; blocks of 128 would keep 36 SMs idle).  The
//     tensor map's box is R rows high; the tile's other rows multiply what shared memory holds and are not read.
//   - a stage holds the same columns of BOTH weights of a gated projection, multiplied into neighbouring accumulators
//     (kept in fp32 / int32 until the gate is applied), so x is read once and the product needs no second kernel.
//
// Where even shares would be narrow, K is split over the CTAs of a cluster instead (2 or 4): a CTA then streams up to
// four times the columns over a part of K, reads that part of x only, and wastes less of the 128-row instruction.  The
// partial sums meet in shared memory over the cluster: each CTA takes its share of x's rows, sums the parts in the
// cluster's order (fixed, so the result does not depend on timing; exact in int32) and applies scales and gate.  The
// scales wait in shared memory by then: fetched row by row they were 1 to 2 us of a call (256 x 4096 x 4096 13.6 / 12.9,
// 256 x 1024 x 1024 12.9 / 10.8).
//
//   warp 0     TMA producer            warp 1     MMA issuer (M = 128, N = NM)
//   warps 2-5  epilogue: lane = weight column, registers = rows of x
#include <algorithm>
#include <string>

#include "activation.cuh"
#include "common.cuh"
#include "epilogue.cuh"
#include "host.h"

namespace hb {

namespace {

constexpr int FR_BK = 128;  // bytes of K per stage = one swizzle row
// Epilogue warps: a CTA's last (mostly only) unit ends with all of x's rows times its columns to scale, gate and store,
// and nothing left to hide that behind, so the warps grow with the rows of x.
constexpr int fr_epi_warps(int nm) { return nm <= 16 ? 4 : (nm == 32 ? 8 : 16); }
// What the partial sums of a cluster take in each CTA: splits senders x W weights x NM / splits rows x 128 columns.
constexpr int fr_exchange_bytes(int w, int nm) { return w * nm * 128 * 4; }
constexpr int fr_threads(int nm) { return 64 + 32 * fr_epi_warps(nm); }
constexpr int FR_MAX_STAGES = 32;
constexpr int FR_TILE_BYTES = 128 * FR_BK;  // what one instruction's operand of 128 rows spans
constexpr int FR_SMEM_LIMIT = 227 * 1024;
constexpr int FR_STATIC_BYTES = (2 * FR_MAX_STAGES + 5) * 8 + 16 + 256 * 4;  // barriers and scales

struct FewRowsParams {
  void* out;
  int M, N, K;      // K in bytes
  int rows;         // weight columns per unit (R), a multiple of 8: whole swizzle atoms
  int slabs;        // 128-byte blocks of K per stage
  int splits;       // CTAs of a cluster that share K (1, 2 or 4); above 1 a cluster has one unit
  int stages;
  int act;
  int64_t ldc;
  uint32_t* status;
  const float *scale_x, *scale_w[2];
  int scale_mode;
};

// Maps of `slabs` whole 128-byte blocks of K at once (block, row, 128 bytes) and of one block, whose bytes beyond K
// arrive as zeros.
struct FewRowsMaps {
  CUtensorMap w[2], x;
  CUtensorMap w_tail[2], x_tail;
};

template <int KIND>
__device__ __forceinline__ float to_float(uint32_t acc) {
  return KIND == KIND_S8 ? __int2float_rn(static_cast<int>(acc)) : __uint_as_float(acc);
}

// The scales of weight column n.
template <int W>
__device__ __forceinline__ void load_scales(const FewRowsParams& p, int n, bool live, float (&sw)[W]) {
#pragma unroll
  for (int w = 0; w < W; ++w) {
    sw[w] = p.scale_mode != 0 && live ? __ldg(p.scale_mode == 1 ? p.scale_w[w] : p.scale_w[w] + n) : 1.0f;
  }
}

// The scale of row m of x.
__device__ __forceinline__ float row_scale(const FewRowsParams& p, int m) {
  return p.scale_mode == 0 ? 1.0f : __ldg(p.scale_mode == 1 ? p.scale_x : p.scale_x + m);
}

// Scales, gate, rounding and store of out[m, n].
template <int W, int OUT_DT>
__device__ __forceinline__ void finish(const FewRowsParams& p, int m, int n, float (&v)[W], float sx, const float (&sw)[W]) {
  if (p.scale_mode != 0) {
#pragma unroll
    for (int w = 0; w < W; ++w) v[w] = (v[w] * sx) * sw[w];
  }
  float o = v[0];
  if constexpr (W == 2) o = activate_by<OUT_DT == HB200_DT_FP32>(p.act, v[0]) * v[1];
  const int64_t at = static_cast<int64_t>(m) * p.ldc + n;
  if constexpr (OUT_DT == HB200_DT_FP32) {
    reinterpret_cast<float*>(p.out)[at] = o;
  } else if constexpr (OUT_DT == HB200_DT_BF16) {
    reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o);
  } else {
    reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(o);
  }
}

template <int KIND, int NM, bool GATED, int OUT_DT>
__global__ void __launch_bounds__(fr_threads(NM), 1)
few_rows_kernel(const __grid_constant__ FewRowsMaps maps, const FewRowsParams p) {
  constexpr int W = GATED ? 2 : 1;
  constexpr int ACC_COLS = W * NM;  // one set of accumulators
  constexpr int SUBS = fr_epi_warps(NM) / 4;  // epilogue warps that share a quarter of the columns
  constexpr uint32_t TMEM_COLS = 2 * ACC_COLS < 32 ? 32 : 2 * ACC_COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * FR_MAX_STAGES + 5];
  __shared__ uint32_t misc[2];
  __shared__ float scales_x[NM];  // with K split: those of the block's rows
  const int stages = p.stages;
  uint64_t* full = bars;
  uint64_t* empty = bars + FR_MAX_STAGES;
  uint64_t* acc_full = bars + 2 * FR_MAX_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_full + 4;
  volatile uint32_t* abort_flag = &misc[1];
  const int slab_w = p.rows * FR_BK;             // one weight's share of a block of K
  constexpr int slab_x = NM * FR_BK;
  const int slot_bytes = p.slabs * slab_w;       // one weight's share of a stage
  const int stage_bytes = W * slot_bytes + p.slabs * slab_x;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int units = (p.N + p.rows - 1) / p.rows;
  const int k_blocks = (p.K + FR_BK - 1) / FR_BK;
  // this CTA's blocks of K: all, or its part of the cluster's
  const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0u;
  const int kb_per_split = (k_blocks + p.splits - 1) / p.splits;
  const int kb_begin = min(static_cast<int>(rank) * kb_per_split, k_blocks);
  const int kb_end = min(kb_begin + kb_per_split, k_blocks);
  const int whole = min(p.K / FR_BK, kb_end);  // blocks below this lie wholly inside K
  // with K split, a cluster has one unit of one block of NM rows of x; else all of x's rows are one block
  const int cluster = blockIdx.x / p.splits;
  const int m0 = p.splits > 1 ? cluster / units * NM : 0;
  const int first_unit = p.splits > 1 ? cluster % units : cluster;
  const int unit_step = p.splits > 1 ? units : static_cast<int>(gridDim.x);
  const int block_m = min(p.M - m0, NM);  // its rows of x
  const WaitCtx wctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&maps.w[0]);
    if (GATED) tma_prefetch_desc(&maps.w[1]);
    tma_prefetch_desc(&maps.x);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 32 * fr_epi_warps(NM));
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(&misc[0], TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = misc[0];
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------- TMA producer --------------------------------------------
    if (lane == 0) {
      uint32_t it = 0;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t slab_bytes = static_cast<uint32_t>(W * slab_w + slab_x);
      for (int unit = first_unit; unit < units && ok; unit += unit_step) {
        for (int kb = kb_begin; kb < kb_end; kb += p.slabs, ++it) {
          if (!mbar_wait(&empty[s], ph ^ 1u, wctx, SITE_GEMM_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + s * stage_bytes;
          // rows of the weight maps are columns of the weight; what lies beyond N, M or K arrives as zeros
          if (kb + p.slabs <= whole) {
            mbar_arrive_expect_tx(&full[s], slab_bytes * p.slabs);
#pragma unroll
            for (int w = 0; w < W; ++w) tma_load_3d(dst + w * slot_bytes, &maps.w[w], &full[s], 0, unit * p.rows, kb);
            tma_load_3d(dst + W * slot_bytes, &maps.x, &full[s], 0, m0, kb);
          } else {
            const int blocks = min(p.slabs, kb_end - kb);
            mbar_arrive_expect_tx(&full[s], slab_bytes * blocks);
            for (int b = 0; b < blocks; ++b) {
              const int k = (kb + b) * FR_BK;
#pragma unroll
              for (int w = 0; w < W; ++w) {
                tma_load_2d(dst + w * slot_bytes + b * slab_w, &maps.w_tail[w], &full[s], k, unit * p.rows);
              }
              tma_load_2d(dst + W * slot_bytes + b * slab_x, &maps.x_tail, &full[s], k, m0);
            }
          }
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok) {
        const uint32_t n = static_cast<uint32_t>(stages);
        const uint32_t back = it < n ? it : n;
        for (uint32_t j = it - back; j < it; ++j) mbar_drain(&full[j % n], (j / n) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------- MMA issuer ----------------------------------------------
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc<KIND>(128, NM, false, false);
      int s = 0;
      uint32_t ph = 0;
      uint32_t unit_iter = 0;
      bool ok = true;
      for (int unit = first_unit; unit < units && ok; unit += unit_step, ++unit_iter) {
        const uint32_t acc = unit_iter & 1u;
        const uint32_t acc_ph = (unit_iter >> 1) & 1u;
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, wctx, SITE_GEMM_ACC_EMPTY)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * ACC_COLS;
        for (int kb = kb_begin; kb < kb_end; kb += p.slabs) {
          if (!mbar_wait(&full[s], ph, wctx, SITE_GEMM_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t w_addr = smem_u32(smem + s * stage_bytes);
          // K-major operands: 128-byte rows, 8-row swizzle atoms 1024 bytes apart
          const int blocks = min(p.slabs, kb_end - kb);
          for (int b = 0; b < blocks; ++b) {
            const uint64_t x_desc = make_smem_desc(w_addr + W * slot_bytes + b * slab_x, 16, 1024, SWZ_128B);
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const uint64_t w_desc = make_smem_desc(w_addr + w * slot_bytes + b * slab_w, 16, 1024, SWZ_128B);
#pragma unroll
              for (int k = 0; k < FR_BK / 32; ++k) {
                umma_ss<KIND>(d_tmem + w * NM, desc_advance(w_desc, k * 32), desc_advance(x_desc, k * 32), idesc,
                              kb != kb_begin || (b | k) != 0 ? 1u : 0u);
              }
            }
          }
          umma_commit(&empty[s]);
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) umma_commit(&acc_full[acc]);
      }
      if (!ok) {
        umma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
    __syncwarp();
  } else if (p.splits == 1) {
    // ------------------------------- epilogue ------------------------------------------------
    const int quarter = warp & 3;  // a warp may only touch TMEM lanes [32*(warp%4), +32)
    const int mine = quarter * 32 + lane;
    const int sub = (warp - 2) >> 2;
    uint32_t unit_iter = 0;
    for (int unit = first_unit; unit < units; unit += unit_step, ++unit_iter) {
      const uint32_t acc = unit_iter & 1u;
      const uint32_t acc_ph = (unit_iter >> 1) & 1u;
      bool ok = mbar_wait(&acc_full[acc], acc_ph, wctx, SITE_GEMM_ACC_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const int n = unit * p.rows + mine;
      const bool live = mine < p.rows && n < p.N;
      float sw[W];
      load_scales<W>(p, n, live, sw);
      const uint32_t t_row = tmem_base + acc * ACC_COLS + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = sub * 16; c < NM; c += SUBS * 16) {
        if (c >= p.M) break;
        uint32_t r[W][16];
#pragma unroll
        for (int w = 0; w < W; ++w) tmem_ld_32x32b_x16(t_row + w * NM + c, r[w]);
        tmem_wait_ld();
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (c + i < p.M) {
              float v[W];
#pragma unroll
              for (int w = 0; w < W; ++w) v[w] = to_float<KIND>(r[w][i]);
              finish<W, OUT_DT>(p, c + i, n, v, row_scale(p, c + i), sw);
            }
          }
        }
      }
      tc_fence_before_sync();
      mbar_arrive(&acc_empty[acc]);
    }
  }

  if (p.splits > 1) {
    // ------------------------------- partial sums over the cluster ----------------------------
    // Row m of x belongs to CTA (m / 4) % splits.  Every CTA hands the others their rows' partial sums in groups of
    // four, into the ring of stages, which is free once every CTA of the cluster has seen its own products end.
    const int quarter = warp & 3;
    const int mine = quarter * 32 + lane;
    const int sub = (warp - 2) >> 2;
    // the scales are fetched while the products run
    const int n = first_unit * p.rows + mine;
    const bool live = mine < p.rows && n < p.N;
    float sw[W];
    bool ok = true;
    if (warp >= 2) {
      load_scales<W>(p, n, live, sw);
      for (int m = threadIdx.x - 64; m < block_m; m += fr_threads(NM) - 64) scales_x[m] = row_scale(p, m0 + m);
      ok = mbar_wait(acc_full, 0, wctx, SITE_GEMM_ACC_FULL);
      ok = __all_sync(0xffffffffu, ok);
    }
    cluster_sync_all();
    const int groups = (block_m + 3) / 4;
    // slot of (sender, weight, the receiver's j-th group): 128 columns of 16 bytes; a receiver has NM / 4 / splits
    // groups, so all of it is fr_exchange_bytes(W, NM)
    const int held = NM / 4 / p.splits;
    auto slot = [&](int from, int w, int j) { return static_cast<uint32_t>((from * W + w) * held + j) * 2048u + mine * 16u; };
    if (warp >= 2 && ok && quarter * 32 < p.rows) {  // columns that the unit does not have stay here
      tc_fence_after_sync();
      const bool none = kb_begin >= kb_end;  // this CTA had no part of K: its accumulators were never written
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = sub * 16; c < NM; c += SUBS * 16) {
        if (c >= block_m) break;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(t_row + w * NM + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int g = c / 4 + q;
            if (g < groups && mine < p.rows) {
              const uint32_t v[4] = {none ? 0u : r[4 * q], none ? 0u : r[4 * q + 1], none ? 0u : r[4 * q + 2], none ? 0u : r[4 * q + 3]};
              st_cluster_v4(map_to_cta(smem_u32(smem) + slot(rank, w, g / p.splits), g % p.splits), v);
            }
          }
        }
      }
    }
    cluster_sync_all();
    if (warp >= 2 && ok) {
      for (int g = rank + sub * p.splits; g < groups && live; g += SUBS * p.splits) {
        uint4 part[4];
        float v[4][W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            if (f < p.splits) part[f] = *reinterpret_cast<const uint4*>(smem + slot(f, w, g / p.splits));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t sum = (&part[0].x)[i];
#pragma unroll
            for (int f = 1; f < 4; ++f) {
              if (f < p.splits) {
                const uint32_t more = (&part[f].x)[i];
                sum = KIND == KIND_S8 ? sum + more : __float_as_uint(__uint_as_float(sum) + __uint_as_float(more));
              }
            }
            v[i][w] = to_float<KIND>(sum);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (4 * g + i < block_m) finish<W, OUT_DT>(p, m0 + 4 * g + i, n, v[i], scales_x[4 * g + i], sw);
        }
      }
    }
  }

  // ------------------------------- teardown ----------------------------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// How many clusters of `cluster` CTAs the device runs at once (a B200's SMs come in groups whose sizes are not all
// multiples of 4: 74 clusters of 2, 33 of 4 with a CTA on every SM).
cudaError_t max_clusters(const void* kernel, int cluster, int threads, int smem, int* clusters) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg);
}

// Shares of K: as many as leave a CTA at most 128 columns, with four blocks of K each at least; `at_once`: the CTAs or
// clusters that share the columns of a block of NM rows of x.  Measured at 16 rows of x, N = 4096, int8: K = 14336 in 1 / 2 /
// 4 shares 20.8 / 16.2 / 13.5 us, K = 4096 in 9.3 / 9.1 / 7.2 us.
template <int KIND, int NM, bool GATED, int OUT_DT>
int choose_splits(const FewRowsArgs& a, DeviceCtx* ctx, int* splits, int64_t* at_once) {
  auto kernel = few_rows_kernel<KIND, NM, GATED, OUT_DT>;
  static std::atomic<uint64_t> smem_attr_done{0};
  HB_CUDA_CHECK(set_max_dynamic_smem_once(smem_attr_done, reinterpret_cast<const void*>(kernel),
                                          FR_SMEM_LIMIT - FR_STATIC_BYTES, a.device));
  const int64_t k_blocks = (a.K * kind_bytes(KIND) + FR_BK - 1) / FR_BK;
  const int64_t row_blocks = (a.M + NM - 1) / NM;
  const int64_t column_blocks = (a.N + 127) / 128;
  *splits = 1;
  *at_once = ctx->num_sms;
  for (int s = 2; s <= 4 && k_blocks >= 4 * s; s *= 2) {
    static std::atomic<int> fit[2][64];
    std::atomic<int>& known = fit[s / 4][static_cast<unsigned>(a.device) & 63u];
    int clusters = known.load(std::memory_order_relaxed);
    if (clusters == 0) {
      HB_CUDA_CHECK(max_clusters(reinterpret_cast<const void*>(kernel), s, fr_threads(NM), FR_SMEM_LIMIT - FR_STATIC_BYTES, &clusters));
      known.store(clusters, std::memory_order_relaxed);
    }
    if (column_blocks > clusters / row_blocks) break;
    *splits = s;
    *at_once = clusters / row_blocks;
  }
  return HB200_OK;
}

template <int KIND, int NM, bool GATED, int OUT_DT>
int launch_few_rows_instance(const FewRowsArgs& a, DeviceCtx* ctx) {
  constexpr int W = GATED ? 2 : 1;
  constexpr int ES = kind_bytes(KIND);
  auto kernel = few_rows_kernel<KIND, NM, GATED, OUT_DT>;
  FewRowsParams p;
  p.out = a.out;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.K = static_cast<int>(a.K * ES);
  int64_t at_once = 0;
  if (const int rc = choose_splits<KIND, NM, GATED, OUT_DT>(a, ctx, &p.splits, &at_once); rc != HB200_OK) return rc;
  const int64_t row_blocks = (a.M + NM - 1) / NM;
  if (row_blocks > 1 && p.splits == 1) return set_error(HB200_ERR_BAD_CONFIG, "few rows: more rows of x than one block, and K not split");
  // Even shares of the columns: as few rounds of 128 columns as there must be, over all CTAs or clusters that fit at once.
  const int64_t rounds = (a.N + 128 * at_once - 1) / (128 * at_once);
  p.rows = static_cast<int>((a.N + rounds * at_once - 1) / (rounds * at_once) + 7) / 8 * 8;
  const int slab_bytes = (W * p.rows + NM) * FR_BK;
  // An instruction reads 128 rows from the start of a slot of fewer: past the last stage there has to be room for that.
  const int tail = FR_TILE_BYTES;
  const int budget = FR_SMEM_LIMIT - FR_STATIC_BYTES - 1024 - tail;
  // Several blocks of K a stage: what a stage costs beside its bytes (barriers, one TMA request per operand) is then
  // paid for up to 48 KB.  Measured at 16 x 4096 x 14336, int8, K not split: 1 / 2 / 4 / 8 blocks of 6 KB a stage
  // 40.3 / 28.8 / 23.1 / 20.7 us.
  p.slabs = std::max(1, std::min(8, 48 * 1024 / slab_bytes));
  const int stage_bytes = p.slabs * slab_bytes;
  p.stages = std::min(FR_MAX_STAGES, budget / stage_bytes);
  p.act = a.act;
  p.ldc = a.ldc;
  p.status = ctx->status_dev;
  p.scale_x = a.scale_x;
  p.scale_w[0] = a.scale_w[0];
  p.scale_w[1] = a.scale_w[1];
  p.scale_mode = a.scale_mode;
  const int smem = std::max(p.stages * stage_bytes + tail, fr_exchange_bytes(W, NM)) + 1024;

  FewRowsMaps maps;
  for (int w = 0; w < 3; ++w) {  // the weights, then x
    if (w == 1 && !GATED) {
      maps.w[1] = maps.w[0];
      maps.w_tail[1] = maps.w_tail[0];
      continue;
    }
    const void* base = w < 2 ? a.w[w] : a.x;
    const uint64_t rows = static_cast<uint64_t>(w < 2 ? a.N : a.M);
    const uint64_t ld = static_cast<uint64_t>((w < 2 ? a.ldb[w] : a.lda) * ES);
    const uint32_t box_rows = static_cast<uint32_t>(w < 2 ? p.rows : NM);
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), rows};
    const uint32_t box[2] = {FR_BK, box_rows};
    int rc = encode_tmap_u8(w < 2 ? &maps.w_tail[w] : &maps.x_tail, base, 2, dims, &ld, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != HB200_OK) return rc;
    if (p.K < FR_BK) {  // no whole block: the maps of several are not used
      (w < 2 ? maps.w[w] : maps.x) = w < 2 ? maps.w_tail[w] : maps.x_tail;
      continue;
    }
    const uint64_t dims3[3] = {FR_BK, rows, static_cast<uint64_t>(p.K / FR_BK)};
    const uint64_t strides3[2] = {ld, FR_BK};
    const uint32_t box3[3] = {FR_BK, box_rows, static_cast<uint32_t>(p.slabs)};
    rc = encode_tmap_u8(w < 2 ? &maps.w[w] : &maps.x, base, 3, dims3, strides3, box3, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != HB200_OK) return rc;
  }

  const int64_t units = (a.N + p.rows - 1) / p.rows;
  if (p.splits > 1) {
    HB_CUDA_CHECK(launch_pdl_cluster(kernel, static_cast<unsigned>(row_blocks * units * p.splits), fr_threads(NM), p.splits, smem, a.stream, maps, p));
  } else {
    HB_CUDA_CHECK(launch_pdl(kernel, static_cast<unsigned>(std::min<int64_t>(units, ctx->num_sms)), fr_threads(NM), smem, a.stream,
                             maps, p));
  }
  return HB200_OK;
}

template <int KIND, bool GATED, int OUT_DT>
int launch_few_rows_nm(const FewRowsArgs& a, DeviceCtx* ctx) {
  if (a.M <= 16) return launch_few_rows_instance<KIND, 16, GATED, OUT_DT>(a, ctx);
  if (a.M <= 32) return launch_few_rows_instance<KIND, 32, GATED, OUT_DT>(a, ctx);
  if (a.M <= 64) return launch_few_rows_instance<KIND, 64, GATED, OUT_DT>(a, ctx);
  if constexpr (!GATED) {
    if (a.M > 128) return launch_few_rows_instance<KIND, 256, GATED, OUT_DT>(a, ctx);
  }
  return launch_few_rows_instance<KIND, 128, GATED, OUT_DT>(a, ctx);
}

template <int KIND, bool GATED>
int launch_few_rows_out(const FewRowsArgs& a, DeviceCtx* ctx) {
  switch (a.out_dtype) {
    case HB200_DT_FP16:
      return launch_few_rows_nm<KIND, GATED, HB200_DT_FP16>(a, ctx);
    case HB200_DT_BF16:
      return launch_few_rows_nm<KIND, GATED, HB200_DT_BF16>(a, ctx);
    default:
      return launch_few_rows_nm<KIND, GATED, HB200_DT_FP32>(a, ctx);
  }
}

}  // namespace

FewRowsArgs few_rows_args(const GemmArgs& a) {
  FewRowsArgs f;
  f.x = a.x;
  f.w[0] = a.y;
  f.out = a.out;
  f.M = a.M;
  f.N = a.N;
  f.K = a.K;
  f.lda = a.lda;
  f.ldb[0] = a.ldb;
  f.ldc = a.ldc;
  f.out_dtype = a.out_dtype;
  f.kind = a.kind;
  f.device = a.device;
  f.stream = a.stream;
  f.scale_x = a.scale_a;
  f.scale_w[0] = a.scale_b;
  f.scale_mode = a.scale_mode;
  return f;
}

// Asks the instance that launch_few_rows runs for these arguments, so that the two cannot disagree.
int few_rows_splits(const FewRowsArgs& a, DeviceCtx* ctx, int* splits) {
  int64_t at_once = 0;
  switch (a.out_dtype) {
    case HB200_DT_FP16:
      return choose_splits<KIND_S8, 256, false, HB200_DT_FP16>(a, ctx, splits, &at_once);
    case HB200_DT_BF16:
      return choose_splits<KIND_S8, 256, false, HB200_DT_BF16>(a, ctx, splits, &at_once);
    default:
      return choose_splits<KIND_S8, 256, false, HB200_DT_FP32>(a, ctx, splits, &at_once);
  }
}

int launch_few_rows(const FewRowsArgs& a, DeviceCtx* ctx) {
  if (!a.gated) {
    if (a.kind != KIND_S8) return set_error(HB200_ERR_BAD_DTYPE, "few rows: one weight is built for int8 operands only");
    return launch_few_rows_out<KIND_S8, false>(a, ctx);
  }
  switch (a.kind) {
    case KIND_E4M3:
      return launch_few_rows_out<KIND_E4M3, true>(a, ctx);
    case KIND_S8:
      return launch_few_rows_out<KIND_S8, true>(a, ctx);
    case KIND_F16:
      return launch_few_rows_nm<KIND_F16, true, HB200_DT_FP16>(a, ctx);
    default:
      return launch_few_rows_nm<KIND_BF16, true, HB200_DT_BF16>(a, ctx);
  }
}

}  // namespace hb
