// out = act(x Wg) * (x Wu): choice and launch of the kernels for the gated projection (see gated_gemm.cuh for the
// tensor-core kernel and gemm_few_rows.cu for few rows of x).
#include <algorithm>
#include <string>

#include "gated_gemm.cuh"

namespace hb {

namespace {

template <int KIND, bool B_MN, int BN, int MODE, int OUT_DT>
int launch_forward(const GatedArgs& a, DeviceCtx* ctx) {
  constexpr int ES = kind_bytes(KIND);
  GatedMaps maps;
  int rc = gated_operand_map(&maps.a[0], a.x, false, a.K, a.M, a.lda, ES, 128);
  if (rc != HB200_OK) return rc;
  maps.a[1] = maps.a[0];
  for (int w = 0; w < 2; ++w) {
    rc = gated_operand_map(&maps.b[w], a.w[w], B_MN, a.K, a.F, a.ldb[w], ES, BN / 2);
    if (rc != HB200_OK) return rc;
  }
  rc = gated_out_map(&maps.out[0], a.out, a.M, a.F, a.ldc, OUT_DT == HB200_DT_FP32);
  if (rc != HB200_OK) return rc;
  for (int i = 0; i < 2; ++i) {
    maps.out[1 + i] = maps.out[0];
    if (MODE == MODE_GATED_TRAIN) {
      rc = gated_out_map(&maps.out[1 + i], a.saved[i], a.M, a.F, a.F, true);
      if (rc != HB200_OK) return rc;
    }
  }
  GatedParams p;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.F);
  p.k_blocks = static_cast<int>((a.K * ES + GG_BK - 1) / GG_BK);
  p.splits = 1;
  // 16 row blocks share a pass over the weights (4096 x 4096 x 14336, groups of 4 / 8 / 16 / 32: bf16 684 / 666 / 656 / 657 us,
  // e4m3 377 / 368 / 361 / 361 us; at 2048 rows and below 8 and more are the same)
  p.group_m = 16;
  p.act = a.act;
  p.status = ctx->status_dev;
  p.scale_x = a.scale_x;
  p.scale_w[0] = a.scale_w[0];
  p.scale_w[1] = a.scale_w[1];
  p.scale_mode = a.scale_mode;
  return launch_gated_pair<KIND, false, B_MN, BN, MODE, OUT_DT>(maps, p, ctx, a.device, a.stream);
}

template <int KIND, bool B_MN, int MODE, int OUT_DT>
int launch_forward_tile(const GatedArgs& a, DeviceCtx* ctx) {
  return gated_narrow_tiles(a.M, 2 * a.F, 1, ctx->num_sms) ? launch_forward<KIND, B_MN, 128, MODE, OUT_DT>(a, ctx)
                                                            : launch_forward<KIND, B_MN, 256, MODE, OUT_DT>(a, ctx);
}

template <int KIND>
int launch_forward_8bit(const GatedArgs& a, DeviceCtx* ctx) {
  switch (a.out_dtype) {
    case HB200_DT_FP16:
      return launch_forward_tile<KIND, false, MODE_GATED, HB200_DT_FP16>(a, ctx);
    case HB200_DT_BF16:
      return launch_forward_tile<KIND, false, MODE_GATED, HB200_DT_BF16>(a, ctx);
    default:
      return launch_forward_tile<KIND, false, MODE_GATED, HB200_DT_FP32>(a, ctx);
  }
}

template <int KIND, int OUT_DT>
int launch_forward_16bit(const GatedArgs& a, DeviceCtx* ctx) {
  if (a.saved[0] != nullptr) {
    return a.w_colmajor ? launch_forward_tile<KIND, false, MODE_GATED_TRAIN, OUT_DT>(a, ctx)
                        : launch_forward_tile<KIND, true, MODE_GATED_TRAIN, OUT_DT>(a, ctx);
  }
  return a.w_colmajor ? launch_forward_tile<KIND, false, MODE_GATED, OUT_DT>(a, ctx)
                      : launch_forward_tile<KIND, true, MODE_GATED, OUT_DT>(a, ctx);
}

}  // namespace

int launch_gated(const GatedArgs& a, DeviceCtx* ctx) {
  // Few rows against column-major weights stream the weights; the tensor-core tile of 256 rows would mostly be empty.
  if (a.M <= kFewRowsMax && a.w_colmajor && a.saved[0] == nullptr) {
    FewRowsArgs f;
    f.x = a.x;
    f.out = a.out;
    f.M = a.M;
    f.N = a.F;
    f.K = a.K;
    f.lda = a.lda;
    for (int w = 0; w < 2; ++w) {
      f.w[w] = a.w[w];
      f.ldb[w] = a.ldb[w];
      f.scale_w[w] = a.scale_w[w];
    }
    f.ldc = a.ldc;
    f.out_dtype = a.out_dtype;
    f.kind = a.kind;
    f.gated = true;
    f.act = a.act;
    f.device = a.device;
    f.stream = a.stream;
    f.scale_x = a.scale_x;
    f.scale_mode = a.scale_mode;
    return launch_few_rows(f, ctx);
  }
  switch (a.kind) {
    case KIND_E4M3:
      return launch_forward_8bit<KIND_E4M3>(a, ctx);
    case KIND_S8:
      return launch_forward_8bit<KIND_S8>(a, ctx);
    case KIND_F16:
      return launch_forward_16bit<KIND_F16, HB200_DT_FP16>(a, ctx);
    default:
      return launch_forward_16bit<KIND_BF16, HB200_DT_BF16>(a, ctx);
  }
}

}  // namespace hb
