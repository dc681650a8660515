// Products of few rows (M <= 128) with one or two column-major weights: int8_gemm for a handful of tokens, and the
// gated projection act(x Wg) * (x Wu) for them (e4m3, int8, fp16 or bf16 operands).
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
constexpr int FR_THREADS = 192;
constexpr int FR_EPI_THREADS = 128;
constexpr int FR_MAX_STAGES = 32;
constexpr int FR_TILE_BYTES = 128 * FR_BK;  // what one instruction's operand of 128 rows spans
constexpr int FR_SMEM_LIMIT = 227 * 1024;
constexpr int FR_BAR_BYTES = (2 * FR_MAX_STAGES + 5) * 8 + 16;

struct FewRowsParams {
  void* out;
  int M, N, K;      // K in bytes
  int rows;         // weight columns per unit (R)
  int slot_bytes;   // shared memory of R weight columns: whole swizzle atoms of 8
  int stages;
  int act;
  int64_t ldc;
  uint32_t* status;
  const float *scale_x, *scale_w[2];
  int scale_mode;
};

template <int KIND, int NM, bool GATED, int OUT_DT>
__global__ void __launch_bounds__(FR_THREADS, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap tmap_w0, const __grid_constant__ CUtensorMap tmap_w1,
                const __grid_constant__ CUtensorMap tmap_x, const FewRowsParams p) {
  constexpr int W = GATED ? 2 : 1;
  constexpr int ACC_COLS = W * NM;  // one set of accumulators
  constexpr uint32_t TMEM_COLS = 2 * ACC_COLS < 32 ? 32 : 2 * ACC_COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * FR_MAX_STAGES + 5];
  __shared__ uint32_t misc[2];
  const int stages = p.stages;
  uint64_t* full = bars;
  uint64_t* empty = bars + FR_MAX_STAGES;
  uint64_t* acc_full = bars + 2 * FR_MAX_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_full + 4;
  volatile uint32_t* abort_flag = &misc[1];
  const int stage_bytes = W * p.slot_bytes + NM * FR_BK;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int units = (p.N + p.rows - 1) / p.rows;
  const int k_blocks = (p.K + FR_BK - 1) / FR_BK;
  const WaitCtx wctx{abort_flag, p.status};

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_w0);
    if (GATED) tma_prefetch_desc(&tmap_w1);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], FR_EPI_THREADS);
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
      const uint32_t bytes = static_cast<uint32_t>(W * p.rows + NM) * FR_BK;
      for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          if (!mbar_wait(&empty[s], ph ^ 1u, wctx, SITE_GEMM_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + s * stage_bytes;
          mbar_arrive_expect_tx(&full[s], bytes);
          // rows of the weight maps are columns of the weight; what lies beyond N, M or K arrives as zeros
          tma_load_2d(dst, &tmap_w0, &full[s], kb * FR_BK, unit * p.rows);
          if (GATED) tma_load_2d(dst + p.slot_bytes, &tmap_w1, &full[s], kb * FR_BK, unit * p.rows);
          tma_load_2d(dst + W * p.slot_bytes, &tmap_x, &full[s], kb * FR_BK, 0);
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
      for (int unit = blockIdx.x; unit < units && ok; unit += gridDim.x, ++unit_iter) {
        const uint32_t acc = unit_iter & 1u;
        const uint32_t acc_ph = (unit_iter >> 1) & 1u;
        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, wctx, SITE_GEMM_ACC_EMPTY)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * ACC_COLS;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full[s], ph, wctx, SITE_GEMM_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t w_addr = smem_u32(smem + s * stage_bytes);
          // K-major operands: 128-byte rows, 8-row swizzle atoms 1024 bytes apart
          const uint64_t x_desc = make_smem_desc(w_addr + W * p.slot_bytes, 16, 1024, SWZ_128B);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint64_t w_desc = make_smem_desc(w_addr + w * p.slot_bytes, 16, 1024, SWZ_128B);
#pragma unroll
            for (int k = 0; k < FR_BK / 32; ++k) {
              umma_ss<KIND>(d_tmem + w * NM, desc_advance(w_desc, k * 32), desc_advance(x_desc, k * 32), idesc,
                            (kb | k) != 0 ? 1u : 0u);
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
  } else {
    // ------------------------------- epilogue ------------------------------------------------
    const int quarter = warp & 3;  // a warp may only touch TMEM lanes [32*(warp%4), +32)
    const int mine = quarter * 32 + lane;
    uint32_t unit_iter = 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++unit_iter) {
      const uint32_t acc = unit_iter & 1u;
      const uint32_t acc_ph = (unit_iter >> 1) & 1u;
      bool ok = mbar_wait(&acc_full[acc], acc_ph, wctx, SITE_GEMM_ACC_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      const int n = unit * p.rows + mine;
      const bool live = mine < p.rows && n < p.N;
      float sw[2] = {1.0f, 1.0f};
      if (p.scale_mode != 0 && live) {
#pragma unroll
        for (int w = 0; w < W; ++w) sw[w] = __ldg(p.scale_mode == 1 ? p.scale_w[w] : p.scale_w[w] + n);
      }
      const uint32_t t_row = tmem_base + acc * ACC_COLS + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < NM; c += 16) {
        if (c >= p.M) break;
        uint32_t r[W][16];
#pragma unroll
        for (int w = 0; w < W; ++w) tmem_ld_32x32b_x16(t_row + w * NM + c, r[w]);
        tmem_wait_ld();
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int m = c + i;
            if (m < p.M) {
              const float sx = p.scale_mode == 0 ? 1.0f : __ldg(p.scale_mode == 1 ? p.scale_x : p.scale_x + m);
              float v[W];
#pragma unroll
              for (int w = 0; w < W; ++w) {
                v[w] = KIND == KIND_S8 ? __int2float_rn(static_cast<int>(r[w][i])) : __uint_as_float(r[w][i]);
                if (p.scale_mode != 0) v[w] = (v[w] * sx) * sw[w];
              }
              float o = v[0];
              if constexpr (GATED) o = activate_by(p.act, v[0]) * v[1];
              const int64_t at = static_cast<int64_t>(m) * p.ldc + n;
              if constexpr (OUT_DT == HB200_DT_FP32) {
                reinterpret_cast<float*>(p.out)[at] = o;
              } else if constexpr (OUT_DT == HB200_DT_BF16) {
                reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o);
              } else {
                reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(o);
              }
            }
          }
        }
      }
      tc_fence_before_sync();
      mbar_arrive(&acc_empty[acc]);
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
  // even shares: as few rounds of 128 columns per SM as there must be, the columns spread over all of them
  const int64_t rounds = (a.N + 128ll * ctx->num_sms - 1) / (128ll * ctx->num_sms);
  p.rows = static_cast<int>((a.N + rounds * ctx->num_sms - 1) / (rounds * ctx->num_sms));
  p.slot_bytes = (p.rows + 7) / 8 * 8 * FR_BK;
  const int stage_bytes = W * p.slot_bytes + NM * FR_BK;
  // An instruction reads 128 rows from the start of a slot of fewer: past the last stage there has to be room for that.
  const int tail = FR_TILE_BYTES;
  const int k_blocks = (p.K + FR_BK - 1) / FR_BK;
  p.stages = std::min(std::min(FR_MAX_STAGES, std::max(k_blocks, 2)), (FR_SMEM_LIMIT - FR_BAR_BYTES - 1024 - tail) / stage_bytes);
  p.act = a.act;
  p.ldc = a.ldc;
  p.status = ctx->status_dev;
  p.scale_x = a.scale_x;
  p.scale_w[0] = a.scale_w[0];
  p.scale_w[1] = a.scale_w[1];
  p.scale_mode = a.scale_mode;
  const int smem = p.stages * stage_bytes + tail + 1024;

  CUtensorMap tw[2], tx;
  for (int w = 0; w < W; ++w) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(a.N)};
    const uint64_t strides[1] = {static_cast<uint64_t>(a.ldb[w] * ES)};
    const uint32_t box[2] = {FR_BK, static_cast<uint32_t>(p.rows)};
    const int rc = encode_tmap_u8(&tw[w], a.w[w], 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != HB200_OK) return rc;
  }
  if (!GATED) tw[1] = tw[0];
  const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(a.M)};
  const uint64_t strides[1] = {static_cast<uint64_t>(a.lda * ES)};
  const uint32_t box[2] = {FR_BK, NM};
  const int rc = encode_tmap_u8(&tx, a.x, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != HB200_OK) return rc;

  static std::atomic<uint64_t> smem_attr_done{0};
  HB_CUDA_CHECK(set_max_dynamic_smem_once(smem_attr_done, reinterpret_cast<const void*>(kernel),
                                          FR_SMEM_LIMIT - FR_BAR_BYTES, a.device));
  const int64_t units = (a.N + p.rows - 1) / p.rows;
  HB_CUDA_CHECK(launch_pdl(kernel, static_cast<unsigned>(std::min<int64_t>(units, ctx->num_sms)), FR_THREADS, smem, a.stream,
                           tw[0], tw[1], tx, p));
  return HB200_OK;
}

template <int KIND, bool GATED, int OUT_DT>
int launch_few_rows_nm(const FewRowsArgs& a, DeviceCtx* ctx) {
  if (a.M <= 16) return launch_few_rows_instance<KIND, 16, GATED, OUT_DT>(a, ctx);
  if (a.M <= 32) return launch_few_rows_instance<KIND, 32, GATED, OUT_DT>(a, ctx);
  if (a.M <= 64) return launch_few_rows_instance<KIND, 64, GATED, OUT_DT>(a, ctx);
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

int launch_few_rows(const FewRowsArgs& a, DeviceCtx* ctx) {
  if (!a.gated) return launch_few_rows_out<KIND_S8, false>(a, ctx);
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
