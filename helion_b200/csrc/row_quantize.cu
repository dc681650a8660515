// Row-wise quantisation to 8 bits, alone (hb200_quantize_rows) or behind a root-mean-square norm with the
// residual's addition (hb200_rms_norm_quantize): what produces the codes and the row scales that the 8-bit
// GEMMs read.
//
//   s = x + residual            (rounded to x's type in residual_out; the norm takes the unrounded fp32 sum)
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)          (quantize_rows: y = x)
//   scale = max|y| / Q,  code = round(y / scale)                 Q = 448 (e4m3) or 127 (int8)
//
// rstd is one factor for the whole row, so max|y| = rstd * max|s w| and code = (s w) * (Q / max|s w|): the sum of
// squares and the largest magnitude come out of ONE pass and one block reduction, and rstd does not enter the
// codes at all.  All of this is fp32; the codes and residual_out are the only roundings to fewer bits.
//
// Bound by memory: x (and residual) in, residual_out and one byte a value out.  One CTA takes one row; its values
// stay in registers between the reduction and the codes, so global memory is touched once.  Rows longer than
// 1024 threads x 4 groups of 8 are read twice instead (the second time from the L2).
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host.h"

namespace hb {

namespace {

struct RowQuantArgs {
  const void* x;
  const void* residual;  // null: none
  const void* weight;
  void* codes;
  float* scales;
  void* residual_out;
  int64_t N, x_rs, residual_rs, codes_rs, residual_out_rs;
  float inv_n, eps;
  bool weight_fp32;  // else of x's type
  bool int8;         // else e4m3
};

// How a row's groups of 8 values are addressed.
enum RowTier : int {
  ROW_ALIGNED = 0,  // every group of every tensor is whole and aligned to its vector width
  ROW_PHASED = 1,   // rows of any length, but all tensors' rows start at the same place modulo 8 values: the groups
                    // are cut at that common boundary, so all but a row's first and last group are whole vectors
  ROW_SCALAR = 2,   // anything else: value by value
};

constexpr uint32_t kF32AbsMask = 0x7fffffffu;
// Rows whose largest |s w| is below this are rows of zeros (Q / max could overflow).
constexpr float kZeroRow = 7.888609e-31f;  // 2^-100

template <int SRC_DT>
struct Src;
template <>
struct Src<HB200_DT_FP16> {
  using T = __half;
  __device__ static float get(const T* p) { return __half2float(*p); }
  __device__ static T put(float v) { return __float2half_rn(v); }
  __device__ static float2 get2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  __device__ static uint32_t put2(float a, float b) { return pack_f16x2(a, b); }
};
template <>
struct Src<HB200_DT_BF16> {
  using T = __nv_bfloat16;
  __device__ static float get(const T* p) { return __bfloat162float(*p); }
  __device__ static T put(float v) { return __float2bfloat16_rn(v); }
  __device__ static float2 get2(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
  __device__ static uint32_t put2(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Src<HB200_DT_FP32> {
  using T = float;
  __device__ static float get(const T* p) { return *p; }
  __device__ static T put(float v) { return v; }
};

// Eight values from an aligned address.
template <int SRC_DT>
__device__ __forceinline__ void load8(const typename Src<SRC_DT>::T* p, float (&v)[8]) {
  if constexpr (SRC_DT == HB200_DT_FP32) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Src<SRC_DT>::get2(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <int SRC_DT>
__device__ __forceinline__ void store8(typename Src<SRC_DT>::T* p, const float (&v)[8]) {
  if constexpr (SRC_DT == HB200_DT_FP32) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(Src<SRC_DT>::put2(v[0], v[1]), Src<SRC_DT>::put2(v[2], v[3]),
                                              Src<SRC_DT>::put2(v[4], v[5]), Src<SRC_DT>::put2(v[6], v[7]));
  }
}

// Values [lo, lo + 8) of a row of N; those outside the row read as zero and are not written.
template <int SRC_DT, int TIER>
__device__ __forceinline__ void load_group(const typename Src<SRC_DT>::T* row, int64_t lo, int64_t N, float (&v)[8]) {
  if (TIER == ROW_ALIGNED || (TIER == ROW_PHASED && lo >= 0 && lo + 8 <= N)) {
    load8<SRC_DT>(row + lo, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (lo + i >= 0 && lo + i < N) ? Src<SRC_DT>::get(row + lo + i) : 0.0f;
  }
}

// Values [lo, lo + 8) of the weight, whose rows of groups need not be aligned with x's.
template <int W_DT, int TIER>
__device__ __forceinline__ void load_weight(const void* weight, int64_t lo, int64_t N, float (&v)[8]) {
  const auto* w = reinterpret_cast<const typename Src<W_DT>::T*>(weight);
  load_group<W_DT, TIER == ROW_ALIGNED ? ROW_ALIGNED : ROW_SCALAR>(w, lo, N, v);
}

template <int SRC_DT, int TIER>
__device__ __forceinline__ void store_group(typename Src<SRC_DT>::T* row, int64_t lo, int64_t N, const float (&v)[8]) {
  if (TIER == ROW_ALIGNED || (TIER == ROW_PHASED && lo >= 0 && lo + 8 <= N)) {
    store8<SRC_DT>(row + lo, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (lo + i >= 0 && lo + i < N) row[lo + i] = Src<SRC_DT>::put(v[i]);
    }
  }
}

// Round to nearest even.  |v| <= Q up to one rounding; a NaN becomes the NaN code (e4m3) or 0 (int8).
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, bool int8) {
  if (!int8) return pack_e4m3x4(a, b, c, d);
  const uint32_t lo = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040);
  const uint32_t hi = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

template <int TIER>
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t lo, int64_t N, const float (&t)[8], float f, bool int8) {
  const uint32_t a = code4(t[0] * f, t[1] * f, t[2] * f, t[3] * f, int8);
  const uint32_t b = code4(t[4] * f, t[5] * f, t[6] * f, t[7] * f, int8);
  if (TIER == ROW_ALIGNED || (TIER == ROW_PHASED && lo >= 0 && lo + 8 <= N)) {
    *reinterpret_cast<uint2*>(row + lo) = make_uint2(a, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (lo + i >= 0 && lo + i < N) row[lo + i] = static_cast<uint8_t>((i < 4 ? a : b) >> (8 * (i & 3)));
    }
  }
}

// VPT groups of 8 values a thread (0: any number, the row is read twice).  MODE 0: quantise; 1: norm first;
// 2: norm with the residual's addition.
template <int SRC_DT, int VPT, int MODE, int TIER>
__global__ void __launch_bounds__(1024) row_quantize_kernel(RowQuantArgs a) {
  using T = typename Src<SRC_DT>::T;
  constexpr int HELD = VPT > 0 ? VPT : 1;
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_rs;
  const T* r = MODE == 2 ? reinterpret_cast<const T*>(a.residual) + row * a.residual_rs : nullptr;
  T* s_out = MODE == 2 ? reinterpret_cast<T*>(a.residual_out) + row * a.residual_out_rs : nullptr;
  uint8_t* codes = reinterpret_cast<uint8_t*>(a.codes) + row * a.codes_rs;
  // first value of group 0: at or before the row's start
  const int64_t first = TIER == ROW_PHASED ? -static_cast<int64_t>((reinterpret_cast<uintptr_t>(codes)) & 7u) : 0;
  const int64_t groups = (a.N - first + 7) / 8;

  pdl_wait();
  pdl_launch_dependents();

  // s w (or x) of group g; adds to the sum of squares and the largest magnitude, writes the residual sum
  auto take = [&](int64_t g, float (&t)[8], float& sum, uint32_t& top, bool write_sum) {
    const int64_t lo = first + g * 8;
    load_group<SRC_DT, TIER>(x, lo, a.N, t);
    if constexpr (MODE == 2) {
      float rv[8];
      load_group<SRC_DT, TIER>(r, lo, a.N, rv);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] += rv[i];
      if (write_sum) store_group<SRC_DT, TIER>(s_out, lo, a.N, t);
    }
    if constexpr (MODE != 0) {
      float wv[8];
      if (SRC_DT != HB200_DT_FP32 && a.weight_fp32) load_weight<HB200_DT_FP32, TIER>(a.weight, lo, a.N, wv);
      else load_weight<SRC_DT, TIER>(a.weight, lo, a.N, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(t[i], t[i], sum);
        t[i] *= wv[i];
      }
    }
    // magnitudes compared as bit patterns: a NaN is larger than everything and is not lost
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(t[i]) & kF32AbsMask);
  };

  float t[HELD][8];
  float sum = 0.0f;
  uint32_t top = 0;
  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t g = threadIdx.x + static_cast<int64_t>(v) * blockDim.x;
      if (g < groups) take(g, t[v], sum, top, true);
    }
  } else {
    for (int64_t g = threadIdx.x; g < groups; g += blockDim.x) take(g, t[0], sum, top, false);
  }

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (MODE != 0) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (warps > 1) {
    if (lane == 0) {
      red_sum[warp] = sum;
      red_max[warp] = top;
    }
    __syncthreads();
    sum = lane < warps ? red_sum[lane] : 0.0f;
    top = lane < warps ? red_max[lane] : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if constexpr (MODE != 0) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  }

  const float Q = a.int8 ? 127.0f : 448.0f;
  constexpr float kTiny = 1.17549435e-38f;
  const float amax = __uint_as_float(top);
  float rstd = 1.0f;
  if constexpr (MODE != 0) {
    // a sum of squares beyond fp32 (or one that holds an infinity or a NaN) makes the row's scale NaN
    rstd = sum <= 3.402823466e38f ? 1.0f / sqrtf(sum * a.inv_n + a.eps) : __uint_as_float(0x7fc00000u);
  }
  float scale = amax * rstd / Q;
  float f = Q / amax;
  if (amax < kZeroRow || scale < kTiny) {
    scale = kTiny;
    f = 0.0f;
  }
  if (threadIdx.x == 0) a.scales[row] = scale;

  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t g = threadIdx.x + static_cast<int64_t>(v) * blockDim.x;
      if (g < groups) store_codes<TIER>(codes, first + g * 8, a.N, t[v], f, a.int8);
    }
  } else {
    for (int64_t g = threadIdx.x; g < groups; g += blockDim.x) {
      float s2 = 0.0f;
      uint32_t t2 = 0;
      take(g, t[0], s2, t2, true);
      store_codes<TIER>(codes, first + g * 8, a.N, t[0], f, a.int8);
    }
  }
}

template <int SRC_DT, int VPT, int MODE, int TIER>
int launch_row(const RowQuantArgs& a, int64_t M, int threads, cudaStream_t stream) {
  HB_CUDA_CHECK(launch_pdl(row_quantize_kernel<SRC_DT, VPT, MODE, TIER>, static_cast<unsigned>(M),
                           static_cast<unsigned>(threads), 0, stream, a));
  return HB200_OK;
}

template <int SRC_DT, int MODE, int TIER>
int launch_row_size(const RowQuantArgs& a, int64_t M, cudaStream_t stream) {
  const int64_t groups = (a.N + (TIER == ROW_PHASED ? 7 : 0) + 7) / 8;  // a phase adds a group at most
  const int vpt = groups <= 512 ? 1 : (groups <= 1024 ? 2 : 4);
  const int threads = static_cast<int>(std::min<int64_t>(((groups + vpt - 1) / vpt + 31) / 32 * 32, 1024));
  if constexpr (TIER != ROW_SCALAR) {
    if (groups <= 4096) {
      if (vpt == 1) return launch_row<SRC_DT, 1, MODE, TIER>(a, M, threads, stream);
      if (vpt == 2) return launch_row<SRC_DT, 2, MODE, TIER>(a, M, threads, stream);
      return launch_row<SRC_DT, 4, MODE, TIER>(a, M, threads, stream);
    }
  }
  return launch_row<SRC_DT, 0, MODE, TIER>(a, M, threads, stream);
}

// `at` modulo 8 values, or -1 for an address that is not a multiple of the value's size.
int phase_of(const void* at, int elem) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(at);
  return p % elem != 0 ? -1 : static_cast<int>((p / elem) % 8);
}

// Whether every row starts at a 16-byte boundary (8 bytes for codes, whose groups are 8 bytes).
bool rows_aligned(const void* at, int64_t rs, int elem) {
  const uintptr_t bytes = elem == 1 ? 8 : 16;
  return reinterpret_cast<uintptr_t>(at) % bytes == 0 && (static_cast<uintptr_t>(rs) * elem) % bytes == 0;
}

RowTier pick_tier(const RowQuantArgs& a, int mode, int elem, int w_elem) {
  const bool res = mode == 2;
  bool aligned = a.N % 8 == 0 && rows_aligned(a.x, a.x_rs, elem) && rows_aligned(a.codes, a.codes_rs, 1);
  if (res) aligned = aligned && rows_aligned(a.residual, a.residual_rs, elem) && rows_aligned(a.residual_out, a.residual_out_rs, elem);
  if (mode != 0) aligned = aligned && rows_aligned(a.weight, 0, w_elem);
  if (aligned) return ROW_ALIGNED;
  const int64_t step = a.codes_rs & 7;
  bool phased = phase_of(a.x, elem) == phase_of(a.codes, 1) && (a.x_rs & 7) == step;
  if (res) {
    phased = phased && phase_of(a.residual, elem) == phase_of(a.codes, 1) && (a.residual_rs & 7) == step &&
             phase_of(a.residual_out, elem) == phase_of(a.codes, 1) && (a.residual_out_rs & 7) == step;
  }
  return phased ? ROW_PHASED : ROW_SCALAR;
}

template <int SRC_DT, int MODE>
int launch_row_tier(const RowQuantArgs& a, int64_t M, cudaStream_t stream) {
  constexpr int elem = sizeof(typename Src<SRC_DT>::T);
  switch (pick_tier(a, MODE, elem, a.weight_fp32 ? 4 : elem)) {
    case ROW_ALIGNED:
      return launch_row_size<SRC_DT, MODE, ROW_ALIGNED>(a, M, stream);
    case ROW_PHASED:
      return launch_row_size<SRC_DT, MODE, ROW_PHASED>(a, M, stream);
    default:
      return launch_row_size<SRC_DT, MODE, ROW_SCALAR>(a, M, stream);
  }
}

template <int SRC_DT>
int launch_row_mode(const RowQuantArgs& a, int64_t M, cudaStream_t stream) {
  if (a.weight == nullptr) return launch_row_tier<SRC_DT, 0>(a, M, stream);
  return a.residual == nullptr ? launch_row_tier<SRC_DT, 1>(a, M, stream) : launch_row_tier<SRC_DT, 2>(a, M, stream);
}

}  // namespace

int launch_row_quantize(const RowQuantCall& c, cudaStream_t stream) {
  RowQuantArgs a;
  a.x = c.x;
  a.residual = c.residual;
  a.weight = c.weight;
  a.codes = c.codes;
  a.scales = c.scales;
  a.residual_out = c.residual_out;
  a.N = c.N;
  a.x_rs = c.x_rs;
  a.residual_rs = c.residual_rs;
  a.codes_rs = c.codes_rs;
  a.residual_out_rs = c.residual_out_rs;
  a.inv_n = 1.0f / static_cast<float>(c.N);
  a.eps = c.eps;
  a.weight_fp32 = c.weight_dtype == HB200_DT_FP32;
  a.int8 = c.out_dtype == HB200_DT_INT8;
  switch (c.src_dtype) {
    case HB200_DT_FP16:
      return launch_row_mode<HB200_DT_FP16>(a, c.M, stream);
    case HB200_DT_BF16:
      return launch_row_mode<HB200_DT_BF16>(a, c.M, stream);
    default:
      return launch_row_mode<HB200_DT_FP32>(a, c.M, stream);
  }
}

}  // namespace hb
