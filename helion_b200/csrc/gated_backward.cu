// Gradients of h = act(x Wg) * (x Wu) for fp16 / bf16 operands, from dh and what the forward pass kept:
//
//   P = u act'(g),  A = act(g)                       (fp32, written by the forward kernel's epilogue)
//   dG = dh P,  dU = dh A                            one elementwise pass, rounded once to the operands' type: they are
//                                                    operands of the tensor-core products below
//                                                    (fp16: times a power of two where they leave its range, see below)
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

// fp16 holds magnitudes from 2^-24 to 65504, and dG and dU may lie beyond where the gradients do not (under a loss scale, or
// with weights far from 1).  So the elementwise pass also finds the largest finite |dG|, |dU|; if fp16 would lose it or what
// lies 2^-8 below it to its subnormals, both are computed once more times the power of two that puts it into [2^14, 2^15), and
// the products' epilogues divide it out of their fp32 sums.  One factor for both, since dx sums over them.  Ordinary gradients
// are stored once and unscaled; a pass then costs the launch that looks (forward and backward at 333 x 1000 x 2728: 46.6 us, with it 48.3 us).
constexpr float kRangeTop = 65504.0f;
constexpr float kRangeBottom = 0.015625f;  // 2^-6
constexpr int kRangeHead = 32;             // floats before the CTAs' maxima; the first is the factor for the epilogues

// Eight 16-bit values times eight floats (times `scale`), rounded.  `top`: the largest finite magnitude seen, as bits.
template <int DT, bool SCALED>
__device__ __forceinline__ uint4 times8(const uint4& d, const float4& lo, const float4& hi, float scale, uint32_t& top) {
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
  const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 v;
    if constexpr (DT == HB200_DT_FP16) v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    else v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    v.x *= f[2 * j];
    v.y *= f[2 * j + 1];
    if constexpr (SCALED) {
      v.x *= scale;
      v.y *= scale;
    } else if constexpr (DT == HB200_DT_FP16) {
      const uint32_t x = __float_as_uint(v.x) & 0x7fffffffu, y = __float_as_uint(v.y) & 0x7fffffffu;
      top = max(top, max(x < 0x7f800000u ? x : 0u, y < 0x7f800000u ? y : 0u));
    }
    o[j] = DT == HB200_DT_FP16 ? pack_f16x2(v.x, v.y) : pack_bf16x2(v.x, v.y);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

struct ProductArgs {
  const void* dh;
  const float *P, *A;
  void *dg, *du;
  int64_t total, groups_per_row, dh_groups;  // in groups of 8 elements
  float* range;                              // fp16: see kRangeHead
};

// dG = dh P, dU = dh A.  Bound by memory: 2 + 8 bytes in and 4 out for every element of dh.  A thread takes UNROLL groups
// of 8 elements a step, all of their loads first.  Returns the thread's largest finite magnitude.
template <int DT, bool SCALED>
__device__ __forceinline__ uint32_t products(const ProductArgs& a, float scale) {
  constexpr int UNROLL = 2;
  const uint4* d_in = reinterpret_cast<const uint4*>(a.dh);
  const float4* p_in = reinterpret_cast<const float4*>(a.P);
  const float4* a_in = reinterpret_cast<const float4*>(a.A);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  uint32_t top = 0;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < a.total; i0 += UNROLL * step) {
    uint4 d[UNROLL];
    float4 p[UNROLL][2], q[UNROLL][2];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t i = i0 + k * step;
      if (i < a.total) {
        // rows of dh may lie apart; the division is left out where they do not
        const int64_t at = a.dh_groups == a.groups_per_row ? i : i / a.groups_per_row * a.dh_groups + i % a.groups_per_row;
        d[k] = __ldcs(d_in + at);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          p[k][j] = __ldcs(p_in + 2 * i + j);
          q[k][j] = __ldcs(a_in + 2 * i + j);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t i = i0 + k * step;
      if (i < a.total) {
        reinterpret_cast<uint4*>(a.dg)[i] = times8<DT, SCALED>(d[k], p[k][0], p[k][1], scale, top);
        reinterpret_cast<uint4*>(a.du)[i] = times8<DT, SCALED>(d[k], q[k][0], q[k][1], scale, top);
      }
    }
  }
  return top;
}

// The largest of all threads' values, in every thread (256 of them).
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  __shared__ uint32_t of_warp[8];
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, of_warp[threadIdx.x & 7]);
}

template <int DT>
__global__ void __launch_bounds__(256) gated_product_kernel(const ProductArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t top = products<DT, false>(a, 1.0f);
  if constexpr (DT == HB200_DT_FP16) {
    const uint32_t all = block_max(top);
    if (threadIdx.x == 0) a.range[kRangeHead + blockIdx.x] = __uint_as_float(all);
  }
}

// fp16: the products once more, scaled, where the largest of the `blocks` maxima asks for it.
__global__ void __launch_bounds__(256) gated_range_kernel(const ProductArgs a, int blocks) {
  pdl_wait();
  pdl_launch_dependents();
  uint32_t top = 0;
  for (int i = threadIdx.x; i < blocks; i += blockDim.x) top = max(top, __float_as_uint(a.range[kRangeHead + i]));
  top = block_max(top);
  const float largest = __uint_as_float(top);
  const bool fits = top == 0 || (largest >= kRangeBottom && largest <= kRangeTop);
  // 2^14 over the largest's power of two, with both it and its inverse normal
  const int e = max(static_cast<int>(top >> 23) - 127, -112);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.range[0] = fits ? 1.0f : __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
  if (!fits) products<HB200_DT_FP16, true>(a, __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23));
}

GatedParams grad_params(int64_t m, int64_t n, int64_t k_elems, const GatedGradArgs& a, DeviceCtx* ctx) {
  GatedParams p;
  p.M = static_cast<int>(m);
  p.N = static_cast<int>(n);
  p.k_blocks = static_cast<int>((k_elems + 63) / 64);
  p.splits = 1;
  p.group_m = 8;
  p.act = 0;
  p.status = ctx->status_dev;
  p.scale_x = a.kind == KIND_F16 ? a.range : nullptr;
  p.scale_w[0] = p.scale_w[1] = nullptr;
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
  return launch_gated_pair<KIND, false, B_MN, BN, MODE, DT>(maps, grad_params(a.M, a.K, a.F, a, ctx), ctx, a.device, a.stream);
}

// CTAs of the elementwise pass at most.
constexpr int64_t gated_product_blocks(int num_sms) { return 8ll * num_sms; }

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
  GatedParams p = grad_params(a.M, a.K, a.F, a, ctx);
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
  return launch_gated_pair<KIND, true, true, BN, MODE_TWIN, DT>(maps, grad_params(m, n, a.M, a, ctx), ctx, a.device, a.stream);
}

template <int KIND, int DT>
int launch_grad(const GatedGradArgs& a, DeviceCtx* ctx) {
  const int64_t elems = a.M * a.F;
  void* const dgu[2] = {a.dgu, static_cast<uint16_t*>(a.dgu) + elems};
  const int64_t blocks = std::min<int64_t>((elems / 8 + 255) / 256, gated_product_blocks(ctx->num_sms));
  const ProductArgs pa{a.dh, a.saved[0], a.saved[1], dgu[0], dgu[1], elems / 8, a.F / 8, a.dh_rs / 8, a.range};
  HB_CUDA_CHECK(launch_pdl(gated_product_kernel<DT>, static_cast<unsigned>(blocks), 256, 0, a.stream, pa));
  if constexpr (DT == HB200_DT_FP16) {
    const int64_t looking = std::min<int64_t>(blocks, 2ll * ctx->num_sms);
    HB_CUDA_CHECK(launch_pdl(gated_range_kernel, static_cast<unsigned>(looking), 256, 0, a.stream, pa, static_cast<int>(blocks)));
  }
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

size_t gated_grad_range_bytes(int num_sms) { return (kRangeHead + gated_product_blocks(num_sms)) * sizeof(float) / 128 * 128 + 128; }

size_t gated_grad_partial_bytes(int64_t M, int64_t F, int64_t K, int num_sms) {
  const int splits = grad_input_splits(M, F, K, num_sms);
  return splits > 1 ? static_cast<size_t>(splits) * M * K * sizeof(float) : 0;
}

int launch_gated_grad(const GatedGradArgs& a, DeviceCtx* ctx) {
  return a.kind == KIND_F16 ? launch_grad<KIND_F16, HB200_DT_FP16>(a, ctx) : launch_grad<KIND_BF16, HB200_DT_BF16>(a, ctx);
}

}  // namespace hb
