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

// Bound by memory: 2 + 8 bytes in and 4 out for every element of dh.
template <int DT>
__global__ void __launch_bounds__(256) gated_product_kernel(const void* dh, const float* P, const float* A, void* dg, void* du,
                                                            int64_t M, int64_t groups_per_row, int64_t dh_rs) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t total = M * groups_per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t row = i / groups_per_row;
    const int64_t at = row * dh_rs + (i - row * groups_per_row) * 8;
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(dh) + at));
    const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
    float4 pv[2], av[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      pv[j] = __ldcs(reinterpret_cast<const float4*>(P) + 2 * i + j);
      av[j] = __ldcs(reinterpret_cast<const float4*>(A) + 2 * i + j);
    }
    const float* pf = reinterpret_cast<const float*>(pv);
    const float* af = reinterpret_cast<const float*>(av);
    uint32_t g[4], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 d;
      if constexpr (DT == HB200_DT_FP16) d = __half22float2(*reinterpret_cast<const __half2*>(&vw[j]));
      else d = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&vw[j]));
      const float g0 = d.x * pf[2 * j], g1 = d.y * pf[2 * j + 1];
      const float u0 = d.x * af[2 * j], u1 = d.y * af[2 * j + 1];
      g[j] = DT == HB200_DT_FP16 ? pack_f16x2(g0, g1) : pack_bf16x2(g0, g1);
      u[j] = DT == HB200_DT_FP16 ? pack_f16x2(u0, u1) : pack_bf16x2(u0, u1);
    }
    reinterpret_cast<uint4*>(dg)[i] = make_uint4(g[0], g[1], g[2], g[3]);
    reinterpret_cast<uint4*>(du)[i] = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

GatedParams grad_params(int64_t m, int64_t n, int64_t k_elems, DeviceCtx* ctx) {
  GatedParams p;
  p.M = static_cast<int>(m);
  p.N = static_cast<int>(n);
  p.k_blocks = static_cast<int>((k_elems + 63) / 64);
  p.group_m = 8;
  p.act = 0;
  p.status = ctx->status_dev;
  p.scale_x = p.scale_w[0] = p.scale_w[1] = nullptr;
  p.scale_mode = 0;
  return p;
}

// dx [M,K] = dG Wg^T + dU Wu^T: contracted over F, along which a row-major w is contiguous and a column-major one is not.
template <int KIND, int DT, bool B_MN, int BN>
int launch_grad_input(const GatedGradArgs& a, DeviceCtx* ctx, const void* const dgu[2]) {
  GatedMaps maps;
  for (int i = 0; i < 2; ++i) {
    int rc = gated_operand_map(&maps.a[i], dgu[i], false, a.F, a.M, a.F, 2, 128);
    if (rc != HB200_OK) return rc;
    rc = gated_operand_map(&maps.b[i], a.w[i], B_MN, a.F, a.K, a.ldb[i], 2, BN / 2);
    if (rc != HB200_OK) return rc;
  }
  const int rc = gated_out_map(&maps.out[0], a.dx, a.M, a.K, a.K, false);
  if (rc != HB200_OK) return rc;
  maps.out[1] = maps.out[2] = maps.out[0];
  return launch_gated_pair<KIND, false, B_MN, BN, MODE_SUM, DT>(maps, grad_params(a.M, a.K, a.F, ctx), ctx, a.device, a.stream);
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
                           a.saved[1], dgu[0], dgu[1], a.M, a.F / 8, a.dh_rs));
  if (a.dx != nullptr) {
    const bool narrow = gated_narrow_tiles(a.M, a.K, 1, ctx->num_sms);
    int rc;
    if (a.w_colmajor) {
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

int launch_gated_grad(const GatedGradArgs& a, DeviceCtx* ctx) {
  return a.kind == KIND_F16 ? launch_grad<KIND_F16, HB200_DT_FP16>(a, ctx) : launch_grad<KIND_BF16, HB200_DT_BF16>(a, ctx);
}

}  // namespace hb
