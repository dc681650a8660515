// Gradients of h = act(x Wg) * (x Wu) for fp16 / bf16 operands, from dh and what the forward pass kept:
//
//   P = u act'(g),  A = act(g)                       (fp32, written by the forward kernel's epilogue)
//   dG = dh P,  dU = dh A                            one elementwise pass, rounded once to the operands' type: they are
//                                                    operands of the tensor-core products below
//   dx = dG Wg^T + dU Wu^T                           one kernel, its K loop running over both products
//   dWg = x^T dG,  dWu = x^T dU                      one kernel over both products' tiles
//
// The products read every operand where it lies: what a gradient contracts over is the other axis of what the forward
// pass contracted over, so A and B are fed to the tensor cores with their M / N axis contiguous (no transposed copies).
// Keeping P and A rather than g and u moves the activation's work into the forward epilogue, where g and u are still
// exact, and leaves dG and dU with one rounding each.
#include <algorithm>
#include <string>

#include "gated_gemm.cuh"

namespace hb {

namespace {

// Eight 16-bit values times eight floats, rounded.
template <int DT>
__device__ __forceinline__ uint4 times8(const uint4& d, const float4& lo, const float4& hi) {
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
  const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 v;
    if constexpr (DT == HB200_DT_FP16) v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    else v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    o[j] = DT == HB200_DT_FP16 ? pack_f16x2(v.x * f[2 * j], v.y * f[2 * j + 1]) : pack_bf16x2(v.x * f[2 * j], v.y * f[2 * j + 1]);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// dG = dh P, dU = dh A.  Bound by memory: 2 + 8 bytes in and 4 out for every element of dh.  A thread takes UNROLL groups
// of 8 elements a step, all of their loads first.
template <int DT>
__global__ void __launch_bounds__(256) gated_product_kernel(const void* dh, const float* P, const float* A, void* dg, void* du,
                                                            int64_t total, int64_t groups_per_row, int64_t dh_groups) {
  constexpr int UNROLL = 2;
  pdl_wait();
  pdl_launch_dependents();
  const uint4* d_in = reinterpret_cast<const uint4*>(dh);
  const float4* p_in = reinterpret_cast<const float4*>(P);
  const float4* a_in = reinterpret_cast<const float4*>(A);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < total; i0 += UNROLL * step) {
    uint4 d[UNROLL];
    float4 p[UNROLL][2], a[UNROLL][2];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t i = i0 + k * step;
      if (i < total) {
        // rows of dh may lie apart; the division is left out where they do not
        const int64_t at = dh_groups == groups_per_row ? i : i / groups_per_row * dh_groups + i % groups_per_row;
        d[k] = __ldcs(d_in + at);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          p[k][j] = __ldcs(p_in + 2 * i + j);
          a[k][j] = __ldcs(a_in + 2 * i + j);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t i = i0 + k * step;
      if (i < total) {
        reinterpret_cast<uint4*>(dg)[i] = times8<DT>(d[k], p[k][0], p[k][1]);
        reinterpret_cast<uint4*>(du)[i] = times8<DT>(d[k], a[k][0], a[k][1]);
      }
    }
  }
}

GatedParams grad_params(int64_t m, int64_t n, int64_t k_elems, DeviceCtx* ctx) {
  GatedParams p;
  p.M = static_cast<int>(m);
  p.N = static_cast<int>(n);
  p.k_blocks = static_cast<int>((k_elems + 63) / 64);
  p.splits = 1;
  p.group_m = 8;
  p.act = 0;
  p.status = ctx->status_dev;
  p.scale_x = p.scale_w[0] = p.scale_w[1] = nullptr;
  p.scale_mode = 0;
  return p;
}

// dx [M,K] = dG Wg^T + dU Wu^T: contracted over F, along which a row-major w is contiguous and a column-major one is not.
template <int KIND, int DT, bool B_MN, int BN, int MODE = MODE_SUM>
int launch_grad_input(const GatedGradArgs& a, DeviceCtx* ctx, const void* const dgu[2]) {
  GatedMaps maps;
  for (int i = 0; i < 2; ++i) {
    int rc = gated_operand_map(&maps.a[i], dgu[i], false, a.F, a.M, a.F, 2, MODE == MODE_SUM_TALL ? 256 : 128);
    if (rc != HB200_OK) return rc;
    rc = gated_operand_map(&maps.b[i], a.w[i], B_MN, a.F, a.K, a.ldb[i], 2, BN / 2);
    if (rc != HB200_OK) return rc;
  }
  const int rc = gated_out_map(&maps.out[0], a.dx, a.M, a.K, a.K, false);
  if (rc != HB200_OK) return rc;
  maps.out[1] = maps.out[2] = maps.out[0];
  return launch_gated_pair<KIND, false, B_MN, BN, MODE, DT>(maps, grad_params(a.M, a.K, a.F, ctx), ctx, a.device, a.stream);
}

// Units the K loop of dx is cut into: where its tiles leave half of the CTA pairs idle, as many as occupy them, with at
// least eight blocks of K each.
int grad_input_splits(int64_t M, int64_t F, int64_t K, int num_sms) {
  const int64_t tiles = ((M + GG_BM - 1) / GG_BM) * ((K + 255) / 256);
  const int64_t fit = std::min<int64_t>(num_sms / 2 / tiles, 2 * ((F + 63) / 64) / 8);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(fit, 8)));
}

// Tall tiles for dx where they need no more than half the rounds over the CTA pairs that 256-row tiles need.
bool grad_input_tall(int64_t M, int64_t K, int num_sms) {
  const int64_t pairs = num_sms / 2, columns = (K + 255) / 256;
  const int64_t tall = ((M + 511) / 512 * columns + pairs - 1) / pairs;
  const int64_t flat = ((M + 255) / 256 * columns + pairs - 1) / pairs;
  return 2 * tall <= flat;
}

template <int KIND, int DT, bool B_MN>
int launch_grad_input_split(const GatedGradArgs& a, DeviceCtx* ctx, const void* const dgu[2], int splits) {
  GatedMaps maps;
  for (int i = 0; i < 2; ++i) {
    int rc = gated_operand_map(&maps.a[i], dgu[i], false, a.F, a.M, a.F, 2, 128);
    if (rc != HB200_OK) return rc;
    rc = gated_operand_map(&maps.b[i], a.w[i], B_MN, a.F, a.K, a.ldb[i], 2, 128);
    if (rc != HB200_OK) return rc;
  }
  int rc = gated_out_map_layers(&maps.out[0], a.partials, a.M, a.K, splits);
  if (rc != HB200_OK) return rc;
  maps.out[1] = maps.out[2] = maps.out[0];
  GatedParams p = grad_params(a.M, a.K, a.F, ctx);
  // an uneven cut may leave the last units empty: as many as have blocks of K
  const int per = (2 * p.k_blocks + splits - 1) / splits;
  p.splits = (2 * p.k_blocks + per - 1) / per;
  rc = launch_gated_pair<KIND, false, B_MN, 256, MODE_SUM_SPLIT, HB200_DT_FP32>(maps, p, ctx, a.device, a.stream);
  if (rc != HB200_OK) return rc;
  GemmArgs r = {};
  r.M = a.M;
  r.N = a.K;
  r.out = a.dx;
  r.ldc = a.K;
  r.out_dtype = DT;
  r.workspace = a.partials;
  r.stream = a.stream;
  return launch_splitk_reduce(r, p.splits);
}

// Both weights' gradients, contracted over the M tokens: column-major w [F,K] storage dW^T = dG^T x, row-major dW = x^T dG.
template <int KIND, int DT, int BN>
int launch_grad_weights(const GatedGradArgs& a, DeviceCtx* ctx, const void* const dgu[2]) {
  const int64_t m = a.w_colmajor ? a.F : a.K;
  const int64_t n = a.w_colmajor ? a.K : a.F;
  GatedMaps maps;
  for (int i = 0; i < 2; ++i) {
    CUtensorMap* of_x = a.w_colmajor ? &maps.b[i] : &maps.a[i];
    CUtensorMap* of_d = a.w_colmajor ? &maps.a[i] : &maps.b[i];
    int rc = gated_operand_map(of_x, a.x, true, a.M, a.K, a.lda, 2, 0);
    if (rc != HB200_OK) return rc;
    rc = gated_operand_map(of_d, dgu[i], true, a.M, a.F, a.F, 2, 0);
    if (rc != HB200_OK) return rc;
    rc = gated_out_map(&maps.out[i], a.dw[i], m, n, n, false);
    if (rc != HB200_OK) return rc;
  }
  maps.out[2] = maps.out[0];
  return launch_gated_pair<KIND, true, true, BN, MODE_TWIN, DT>(maps, grad_params(m, n, a.M, ctx), ctx, a.device, a.stream);
}

template <int KIND, int DT>
int launch_grad(const GatedGradArgs& a, DeviceCtx* ctx) {
  const int64_t elems = a.M * a.F;
  void* const dgu[2] = {a.dgu, static_cast<uint16_t*>(a.dgu) + elems};
  const int64_t blocks = std::min<int64_t>((elems / 8 + 255) / 256, static_cast<int64_t>(ctx->num_sms) * 8);
  HB_CUDA_CHECK(launch_pdl(gated_product_kernel<DT>, static_cast<unsigned>(blocks), 256, 0, a.stream, a.dh, a.saved[0],
                           a.saved[1], dgu[0], dgu[1], elems / 8, a.F / 8, a.dh_rs / 8));
  if (a.dx != nullptr) {
    const bool narrow = gated_narrow_tiles(a.M, a.K, 1, ctx->num_sms);
    const int splits = grad_input_splits(a.M, a.F, a.K, ctx->num_sms);
    int rc;
    if (splits > 1) {
      rc = a.w_colmajor ? launch_grad_input_split<KIND, DT, true>(a, ctx, dgu, splits)
                        : launch_grad_input_split<KIND, DT, false>(a, ctx, dgu, splits);
    } else if (grad_input_tall(a.M, a.K, ctx->num_sms)) {
      rc = a.w_colmajor ? launch_grad_input<KIND, DT, true, 256, MODE_SUM_TALL>(a, ctx, dgu)
                        : launch_grad_input<KIND, DT, false, 256, MODE_SUM_TALL>(a, ctx, dgu);
    } else if (a.w_colmajor) {
      rc = narrow ? launch_grad_input<KIND, DT, true, 128>(a, ctx, dgu) : launch_grad_input<KIND, DT, true, 256>(a, ctx, dgu);
    } else {
      rc = narrow ? launch_grad_input<KIND, DT, false, 128>(a, ctx, dgu) : launch_grad_input<KIND, DT, false, 256>(a, ctx, dgu);
    }
    if (rc != HB200_OK) return rc;
  }
  if (a.dw[0] != nullptr) {
    const bool narrow = gated_narrow_tiles(a.w_colmajor ? a.F : a.K, a.w_colmajor ? a.K : a.F, 2, ctx->num_sms);
    return narrow ? launch_grad_weights<KIND, DT, 128>(a, ctx, dgu) : launch_grad_weights<KIND, DT, 256>(a, ctx, dgu);
  }
  return HB200_OK;
}

}  // namespace

size_t gated_grad_partial_bytes(int64_t M, int64_t F, int64_t K, int num_sms) {
  const int splits = grad_input_splits(M, F, K, num_sms);
  return splits > 1 ? static_cast<size_t>(splits) * M * K * sizeof(float) : 0;
}

int launch_gated_grad(const GatedGradArgs& a, DeviceCtx* ctx) {
  return a.kind == KIND_F16 ? launch_grad<KIND_F16, HB200_DT_FP16>(a, ctx) : launch_grad<KIND_BF16, HB200_DT_BF16>(a, ctx);
}

}  // namespace hb
