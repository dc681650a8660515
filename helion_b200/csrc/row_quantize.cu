// Row-wise quantisation to 8 bits, alone (hb200_quantize_rows) or behind a root-mean-square norm with the
// residual's addition (hb200_rms_norm_quantize): what produces the codes and the row scales that the 8-bit
// GEMMs read.
//
//   s = x + residual            (rounded to x's type in residual_out; the norm takes the unrounded fp32 sum)
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)          (quantize_rows: y = x)
//   scale = max|y| / Q,  code = round(y Q / max|y|)              Q = 448 (e4m3) or 127 (int8)
//
// rstd is one factor for the whole row, so max|y| = rstd * max|s w| and code = (s w) * (Q / max|s w|): the sum of
// squares and the largest magnitude come out of ONE pass and one block reduction, and rstd does not enter the
// codes at all.  All of this is fp32; the codes and residual_out are the only roundings to fewer bits.
//
// Bound by memory: x (and residual) in, residual_out and one byte a value out.  A CTA takes a row at a time; its values
// stay in registers between the reduction and the codes, so global memory is touched once.  Few rows get a CTA each,
// many rows persistent CTAs fed by bulk copies (row_ring_kernel).  Rows longer than 1024 threads x 4 groups of 8 are read
// twice instead (the second time from the L2).
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
  int64_t M, N, x_rs, residual_rs, codes_rs, residual_out_rs;
  float inv_n, eps;
  bool weight_fp32;     // else of x's type
  bool weight_vectors;  // the weight is 16-byte aligned
  bool int8;            // else e4m3
  bool in_place;        // residual_out is x or the residual
};

struct RowQuantLaunch {
  int64_t M;
  DeviceCtx* ctx;
  int device;
  cudaStream_t stream;
};

// How a row's groups of 8 values are addressed.
enum RowTier : int {
  ROW_ALIGNED = 0,  // every group of every tensor is whole and aligned to its vector width
  ROW_PHASED = 1,   // rows of any length, but all tensors' rows start at the same place modulo 8 values: the groups
                    // are cut at that common boundary, so all but a row's first and last group are whole vectors
  ROW_SCALAR = 2,   // anything else: value by value
};

constexpr uint32_t kF32AbsMask = 0x7fffffffu;
// Rows whose largest |y| is below this are rows of zeros (Q / max|y| may overflow).
constexpr float kZeroRow = 7.888609e-31f;  // 2^-100
// Behind the norm |s w| may be smaller where |y| is not: such a row's values are multiplied by this before the factor.
constexpr float kLift = 18446744073709551616.0f;  // 2^64: the smallest positive |s w|, 2^-149, becomes 2^-85

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
template <int SRC_DT, bool READ_ONLY = false>
__device__ __forceinline__ void load8(const typename Src<SRC_DT>::T* p, float (&v)[8]) {
  if constexpr (SRC_DT == HB200_DT_FP32) {
    const float4* q = reinterpret_cast<const float4*>(p);
    const float4 a = READ_ONLY ? __ldg(q) : q[0], b = READ_ONLY ? __ldg(q + 1) : q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    const uint4 u = READ_ONLY ? __ldg(q) : *q;
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
// [from, to): where the tensor's values lie, relative to the row.  A group that hangs over its row's end, but not over the
// tensor's, is read whole and masked (its other values are a neighbouring row's): a branch to eight single loads
// costs the row's first and last warp a round trip to memory per tensor (1237 x 5003 fp16 with residual: 17.1 us, masked
// 16.0 us).  Not where the sum overwrites x or the residual: another CTA may be writing that neighbouring row.
template <int SRC_DT, int TIER>
__device__ __forceinline__ void load_group(const typename Src<SRC_DT>::T* row, int lo, int N, int from, int to,
                                           float (&v)[8]) {
  if (TIER == ROW_ALIGNED || (TIER == ROW_PHASED && lo >= from && lo + 8 <= to)) {
    load8<SRC_DT>(row + lo, v);
    if constexpr (TIER == ROW_PHASED) {
      if (lo < 0 || lo + 8 > N) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (lo + i >= 0 && lo + i < N) ? v[i] : 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (lo + i >= 0 && lo + i < N) ? Src<SRC_DT>::get(row + lo + i) : 0.0f;
  }
}

// Eight 16-bit values that begin `shift` (1 to 7) values into the 16 of two neighbouring aligned vectors, `aligned` the
// second; without the first its values are zeros.
template <int DT>
__device__ __forceinline__ void load8_shifted(const typename Src<DT>::T* aligned, bool has_first, int shift, float (&v)[8]) {
  const uint4 b = __ldg(reinterpret_cast<const uint4*>(aligned));
  const uint4 a = has_first ? __ldg(reinterpret_cast<const uint4*>(aligned) - 1) : make_uint4(0u, 0u, 0u, 0u);
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  // the shift is the row's, the same in every thread of the CTA
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (shift & 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Src<DT>::get2(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Values [lo, lo + 8) of the weight.  With ROW_PHASED rows lo lies `phase` values before a multiple of 8, where a vector
// of the weight begins: two vectors and a shift instead of eight loads (1237 x 5003 fp16 with residual: 16.0 us, with the
// eight loads, as an fp32 weight has them, 18.9 us).
template <int W_DT, int TIER>
__device__ __forceinline__ void load_weight_as(const void* weight, int lo, int phase, int N, bool vectors, float (&v)[8]) {
  const auto* w = reinterpret_cast<const typename Src<W_DT>::T*>(weight);
  if constexpr (TIER == ROW_PHASED && W_DT != HB200_DT_FP32) {
    const int up = lo + phase;  // a multiple of 8
    if (vectors && up + 8 <= N) {
      if (phase == 0) load8<W_DT, true>(w + lo, v);
      else load8_shifted<W_DT>(w + up, up > 0, 8 - phase, v);
      return;
    }
  }
  if constexpr (TIER == ROW_ALIGNED) {
    load8<W_DT, true>(w + lo, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (lo + i >= 0 && lo + i < N) ? Src<W_DT>::get(w + lo + i) : 0.0f;
  }
}

template <int SRC_DT, int TIER>
__device__ __forceinline__ void load_weight(const RowQuantArgs& a, int lo, int phase, float (&v)[8]) {
  if (SRC_DT != HB200_DT_FP32 && a.weight_fp32) load_weight_as<HB200_DT_FP32, TIER>(a.weight, lo, phase, static_cast<int>(a.N), false, v);
  else load_weight_as<SRC_DT, TIER>(a.weight, lo, phase, static_cast<int>(a.N), a.weight_vectors, v);
}

// Bytes [0, size) of global memory, 16-byte aligned and whole 16-byte pieces, to shared memory.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int SRC_DT, int TIER>
__device__ __forceinline__ void store_group(typename Src<SRC_DT>::T* row, int lo, int N, const float (&v)[8]) {
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

__device__ __forceinline__ void set_pair(float (&v)[8], int i, uint64_t pair) {
  uint32_t a, b;
  unpack2(pair, a, b);
  v[2 * i] = __uint_as_float(a);
  v[2 * i + 1] = __uint_as_float(b);
}

template <int TIER>
__device__ __forceinline__ void store_codes(uint8_t* row, int lo, int N, const float (&t)[8], float2 f, bool int8) {
  float v[8];
  const uint64_t hi = pack2f(f.x, f.x), lo2 = pack2f(f.y, f.y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t t2 = pack2f(t[2 * i], t[2 * i + 1]);
    set_pair(v, i, ffma2(t2, hi, fmul2(t2, lo2)));
  }
  const uint32_t a = code4(v[0], v[1], v[2], v[3], int8);
  const uint32_t b = code4(v[4], v[5], v[6], v[7], int8);
  if (TIER == ROW_ALIGNED || (TIER == ROW_PHASED && lo >= 0 && lo + 8 <= N)) {
    *reinterpret_cast<uint2*>(row + lo) = make_uint2(a, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (lo + i >= 0 && lo + i < N) row[lo + i] = static_cast<uint8_t>((i < 4 ? a : b) >> (8 * (i & 3)));
    }
  }
}

// One row's factor Q / max for the codes, as a sum of two floats, and its scale.  Values of few bits often lie exactly between
// two codes (max / 2 does for int8); the factor's own rounding would decide these ties by chance: with one float 2.734375 in a
// row with the maximum 3.0625 is 400.00003 instead of 400 and gets the code 416 instead of 384.  With two the product is within
// 2^-46 before its rounding to fp32, and every code of 16-bit values is that of the exact quotient.
// `lift`: the values need kLift first.
template <int MODE>
__device__ __forceinline__ float2 row_factor(const RowQuantArgs& a, float sum, uint32_t top, float& scale, bool& lift) {
  const float Q = a.int8 ? 127.0f : 448.0f;
  float amax = __uint_as_float(top);
  float y_max = amax;
  lift = false;
  if constexpr (MODE != 0) {
    // a sum of squares beyond fp32 (or one that holds an infinity or a NaN) makes the row's scale NaN
    y_max *= sum <= 3.402823466e38f ? 1.0f / sqrtf(sum * a.inv_n + a.eps) : __uint_as_float(0x7fc00000u);
    lift = amax < kZeroRow;
    if (lift) amax *= kLift;
  }
  scale = y_max / Q;
  float f = Q / amax;
  if (y_max < kZeroRow) {
    scale = 1.17549435e-38f;
    f = 0.0f;
  }
  return make_float2(f, f > 0.0f ? fmaf(-f, amax, Q) * (f * (a.int8 ? 1.0f / 127.0f : 1.0f / 448.0f)) : 0.0f);
}

__device__ __forceinline__ void lift_group(float (&t)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] *= kLift;
}

// t += r, two values an instruction (the kernels issue close to what an SM can where rows come fast).
__device__ __forceinline__ void add_group(float (&t)[8], const float (&r)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) set_pair(t, i, fadd2(pack2f(t[2 * i], t[2 * i + 1]), pack2f(r[2 * i], r[2 * i + 1])));
}

// Eight values of s w (or x) into the row's sum of squares (as two sums) and largest magnitude; t holds s (or x) on entry.
template <int MODE>
__device__ __forceinline__ void take_group(float (&t)[8], const float (&w)[8], uint64_t& sum2, uint32_t& top) {
  if constexpr (MODE != 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t t2 = pack2f(t[2 * i], t[2 * i + 1]);
      sum2 = ffma2(t2, t2, sum2);
      set_pair(t, i, fmul2(t2, pack2f(w[2 * i], w[2 * i + 1])));
    }
  }
  // magnitudes compared as bit patterns: a NaN is larger than everything and is not lost
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(t[i]) & kF32AbsMask);
}

__device__ __forceinline__ float both(uint64_t sum2) {
  uint32_t a, b;
  unpack2(sum2, a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

template <int MODE>
__device__ __forceinline__ void warp_reduce(float& sum, uint32_t& top) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (MODE != 0) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
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
  const int N = static_cast<int>(a.N);
  const int first = TIER == ROW_PHASED ? -static_cast<int>(reinterpret_cast<uintptr_t>(codes) & 7u) : 0;
  const int groups = (N - first + 7) / 8;
  // how far outside the row its tensors go on, up to a group: rows that may be read too
  auto reach = [&](int64_t rows, int64_t rs) { return a.in_place ? 0 : static_cast<int>(min(rows * rs, int64_t(8))); };
  const int x_before = reach(row, a.x_rs), x_behind = reach(a.M - 1 - row, a.x_rs);
  const int r_before = reach(row, a.residual_rs), r_behind = reach(a.M - 1 - row, a.residual_rs);

  pdl_wait();
  pdl_launch_dependents();

  // x of group g, and the residual
  auto load = [&](int g, float (&t)[8], float (&rv)[8]) {
    load_group<SRC_DT, TIER>(x, first + g * 8, N, -x_before, N + x_behind, t);
    if constexpr (MODE == 2) load_group<SRC_DT, TIER>(r, first + g * 8, N, -r_before, N + r_behind, rv);
  };
  // s w (or x) of group g; adds to the sum of squares and the largest magnitude, writes the residual sum
  auto take = [&](int g, float (&t)[8], const float (&rv)[8], uint64_t& sum2, uint32_t& top, bool write_sum) {
    const int lo = first + g * 8;
    float wv[8];
    if constexpr (MODE != 0) load_weight<SRC_DT, TIER>(a, lo, -first, wv);
    if constexpr (MODE == 2) {
      add_group(t, rv);
      if (write_sum) store_group<SRC_DT, TIER>(s_out, lo, N, t);
    }
    take_group<MODE>(t, wv, sum2, top);
  };

  float t[HELD][8], rv[HELD][8];
  uint64_t sum2 = pack2f(0.0f, 0.0f);
  uint32_t top = 0;
  if constexpr (VPT > 0) {
    // all of a thread's loads before its first store: a store may be to x or the residual itself, so the compiler
    // cannot move a load over one
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int g = threadIdx.x + v * blockDim.x;
      if (g < groups) load(g, t[v], rv[v]);
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int g = threadIdx.x + v * blockDim.x;
      if (g < groups) take(g, t[v], rv[v], sum2, top, true);
    }
  } else {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
      load(g, t[0], rv[0]);
      take(g, t[0], rv[0], sum2, top, false);
    }
  }

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float sum = both(sum2);
  warp_reduce<MODE>(sum, top);
  if (warps > 1) {
    if (lane == 0) {
      red_sum[warp] = sum;
      red_max[warp] = top;
    }
    __syncthreads();
    sum = lane < warps ? red_sum[lane] : 0.0f;
    top = lane < warps ? red_max[lane] : 0u;
    warp_reduce<MODE>(sum, top);
  }
  float scale;
  bool lift;
  const float2 f = row_factor<MODE>(a, sum, top, scale, lift);
  if (threadIdx.x == 0) a.scales[row] = scale;

  if constexpr (VPT > 0) {
    if (MODE != 0 && lift) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) lift_group(t[v]);
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int g = threadIdx.x + v * blockDim.x;
      if (g < groups) store_codes<TIER>(codes, first + g * 8, N, t[v], f, a.int8);
    }
  } else {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
      uint64_t s2 = pack2f(0.0f, 0.0f);
      uint32_t t2 = 0;
      load(g, t[0], rv[0]);
      take(g, t[0], rv[0], s2, t2, true);
      if (MODE != 0 && lift) lift_group(t[0]);
      store_codes<TIER>(codes, first + g * 8, N, t[0], f, a.int8);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Many long 16-bit rows: persistent CTAs whose rows arrive in a ring of shared-memory stages by bulk copies, so that the
// memory system stays busy while a row waits for its reduction.  (With a CTA a row, loads and reductions take turns, and
// the registers of an SM's two to four CTAs hold too few rows in flight.)  A stage is one row of x (and one of the
// residual); values go to registers on arrival, and the reduction's barrier hands the stage back for the row `stages` ahead.
//
// Measured, bf16, a CTA a row / ring (us; % of the copy bandwidth of 6.55 TB/s): with norm and residual 8192 x 4096
// 44.5 / 42.3 (85 %), 4096 x 8192 52.4 / 41.0, 4096 x 14336 93.1 / 68.6 (91 %), 600 x 8192 10.9 / 10.4, but 2048 x 4096
// 13.4 / 15.8; quantised 8192 x 4096 27.6 / 23.0 (67 %), 4096 x 14336 47.0 / 31.9 (84 %), but 600 x 8192 4.2 / 5.4.
// With the norm alone, and for fp32 rows, whose CTAs hold twice the bytes each, it gains nothing (4096 x 8192 with norm
// 29.7 / 32.0; fp32 4096 x 8192 with residual 70.3 / 77.5), nor for rows that are not aligned.
// ------------------------------------------------------------------------------------------------
constexpr int RING_MAX_STAGES = 8;
constexpr int RING_SMEM_PER_SM = 220 * 1024;

struct RowRing {
  int64_t M;
  int stages;
  int row_bytes;  // of one tensor
  uint32_t* status;
};

template <int SRC_DT, int VPT, int MODE>
__global__ void __launch_bounds__(VPT == 2 ? 1024 : 512) row_ring_kernel(RowQuantArgs a, RowRing ring) {
  using T = typename Src<SRC_DT>::T;
  constexpr int TENSORS = MODE == 2 ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[RING_MAX_STAGES];
  __shared__ float red_sum[2][32];
  __shared__ uint32_t red_max[2][32];
  __shared__ uint32_t abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const WaitCtx wctx{abort_flag, ring.status};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int groups = static_cast<int>(a.N / 8);
  const int64_t step = gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ring.stages; ++s) mbar_init(&full[s], 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  auto request = [&](int64_t row, int s) {
    uint8_t* dst = smem + s * TENSORS * ring.row_bytes;
    mbar_arrive_expect_tx(&full[s], TENSORS * ring.row_bytes);
    bulk_load(dst, reinterpret_cast<const T*>(a.x) + row * a.x_rs, ring.row_bytes, &full[s]);
    if constexpr (MODE == 2) {
      bulk_load(dst + ring.row_bytes, reinterpret_cast<const T*>(a.residual) + row * a.residual_rs, ring.row_bytes, &full[s]);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring.stages; ++s) {
      if (blockIdx.x + s * step < ring.M) request(blockIdx.x + s * step, s);
    }
  }

  int s = 0;
  uint32_t ph = 0, turn = 0;
  for (int64_t row = blockIdx.x; row < ring.M; row += step) {
    const T* sx = reinterpret_cast<const T*>(smem + s * TENSORS * ring.row_bytes);
    const bool ok = mbar_wait(&full[s], ph, wctx, SITE_ROWS_FULL);
    float t[VPT][8];
    uint64_t sum2 = pack2f(0.0f, 0.0f);
    uint32_t top = 0;
    if (ok) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int g = threadIdx.x + v * blockDim.x;
        if (g < groups) {
          load8<SRC_DT>(sx + g * 8, t[v]);
          if constexpr (MODE == 2) {
            float rv[8];
            load8<SRC_DT>(sx + ring.row_bytes / sizeof(T) + g * 8, rv);
            add_group(t[v], rv);
            store8<SRC_DT>(reinterpret_cast<T*>(a.residual_out) + row * a.residual_out_rs + g * 8, t[v]);
          }
          float wv[8];
          if constexpr (MODE != 0) load_weight<SRC_DT, ROW_ALIGNED>(a, g * 8, 0, wv);
          take_group<MODE>(t[v], wv, sum2, top);
        }
      }
    }
    float sum = both(sum2);
    warp_reduce<MODE>(sum, top);
    if (lane == 0) {
      red_sum[turn][warp] = sum;
      red_max[turn][warp] = top;
    }
    // every thread has its values of this stage (or a wait ran out: all leave together)
    if (!__syncthreads_and(ok)) break;
    if (threadIdx.x == 0 && row + ring.stages * step < ring.M) request(row + ring.stages * step, s);
    sum = lane < warps ? red_sum[turn][lane] : 0.0f;
    top = lane < warps ? red_max[turn][lane] : 0u;
    warp_reduce<MODE>(sum, top);
    float scale;
    bool lift;
    const float2 f = row_factor<MODE>(a, sum, top, scale, lift);
    if (threadIdx.x == 0) a.scales[row] = scale;
    if (MODE != 0 && lift) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) lift_group(t[v]);
    }
    uint8_t* codes = reinterpret_cast<uint8_t*>(a.codes) + row * a.codes_rs;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int g = threadIdx.x + v * blockDim.x;
      if (g < groups) store_codes<ROW_ALIGNED>(codes, g * 8, 0, t[v], f, a.int8);
    }
    turn ^= 1u;
    if (++s == ring.stages) {
      s = 0;
      ph ^= 1u;
    }
  }
  if (*abort_flag && threadIdx.x == 0) {
    // give copies that are still in flight time to land before shared memory is released
    for (int i = 0; i < ring.stages; ++i) {
      mbar_drain(&full[s], ph);
      if (++s == ring.stages) {
        s = 0;
        ph ^= 1u;
      }
    }
  }
}

template <int SRC_DT, int VPT, int MODE>
int launch_ring(const RowQuantArgs& a, const RowRing& ring, int ctas_per_sm, const RowQuantLaunch& l) {
  auto kernel = row_ring_kernel<SRC_DT, VPT, MODE>;
  static std::atomic<uint64_t> smem_attr_done{0};
  HB_CUDA_CHECK(set_max_dynamic_smem_once(smem_attr_done, reinterpret_cast<const void*>(kernel), RING_SMEM_PER_SM, l.device));
  const int64_t grid = std::min<int64_t>(ring.M, static_cast<int64_t>(l.ctx->num_sms) * ctas_per_sm);
  const int64_t threads = ((a.N / 8 + VPT - 1) / VPT + 31) / 32 * 32;
  HB_CUDA_CHECK(launch_pdl(kernel, static_cast<unsigned>(grid), static_cast<unsigned>(threads),
                           static_cast<size_t>(ring.stages) * ring.row_bytes * (MODE == 2 ? 2 : 1), l.stream, a, ring));
  return HB200_OK;
}

// The ring kernel where it applies (see its measurements): rows of 4096 to 16384 values, enough of them that its CTAs loop.
// Returns 1 where it does not.
template <int SRC_DT, int MODE>
int try_ring(const RowQuantArgs& a, const RowQuantLaunch& l) {
  if (l.M < 4ll * l.ctx->num_sms || a.N < 4096 || a.N > 16384) return 1;
  const int64_t values = l.M * a.N;
  if (MODE == 2 ? a.N < 8192 && values < (1 << 24) : values < (1 << 25)) return 1;
  RowRing ring;
  ring.M = l.M;
  ring.status = l.ctx->status_dev;
  ring.row_bytes = static_cast<int>(a.N) * 2;
  // as many CTAs an SM as have two stages each: 4 of 256 to 512 threads, 2 of up to 512, 1 of up to 1024
  for (int ctas = a.N <= 8192 ? 4 : 2; ctas >= 1; ctas /= 2) {
    ring.stages = std::min(RING_MAX_STAGES, (RING_SMEM_PER_SM / ctas - 2048) / (ring.row_bytes * (MODE == 2 ? 2 : 1)));
    if (ring.stages < 2) continue;
    return ctas == 2 && a.N > 8192 ? launch_ring<SRC_DT, 4, MODE>(a, ring, ctas, l) : launch_ring<SRC_DT, 2, MODE>(a, ring, ctas, l);
  }
  return 1;
}

template <int SRC_DT, int VPT, int MODE, int TIER>
int launch_row(const RowQuantArgs& a, const RowQuantLaunch& l, int threads) {
  HB_CUDA_CHECK(launch_pdl(row_quantize_kernel<SRC_DT, VPT, MODE, TIER>, static_cast<unsigned>(l.M),
                           static_cast<unsigned>(threads), 0, l.stream, a));
  return HB200_OK;
}

template <int SRC_DT, int MODE, int TIER>
int launch_row_size(const RowQuantArgs& a, const RowQuantLaunch& l) {
  const int64_t groups = (a.N + (TIER == ROW_PHASED ? 7 : 0) + 7) / 8;  // a phase adds a group at most
  // CTAs of up to 1024 threads, rather than 512, where a row's own latency counts: rows that have an SM each (one row of
  // 14336 bf16 with residual 4.4 / 3.4 us, quantised 2.4 / 2.2 us), and odd rows with a residual, whose masks and
  // shifts are most of their time (1237 x 5003 17.1 / 15.7 us, 4096 x 4099 47.6 / 39.2 us).  Elsewhere the smaller ones hold
  // more rows a SM (1237 x 8192 quantised 8.0 / 10.5 us).
  const bool wide = l.M <= l.ctx->num_sms || (TIER == ROW_PHASED && MODE == 2 && groups <= 1024);
  const int vpt = groups <= (wide ? 1024 : 512) ? 1 : (groups <= (wide ? 2048 : 1024) ? 2 : 4);
  const int threads = static_cast<int>(std::min<int64_t>(((groups + vpt - 1) / vpt + 31) / 32 * 32, 1024));
  if constexpr (TIER != ROW_SCALAR) {
    if constexpr (TIER == ROW_ALIGNED && MODE != 1 && SRC_DT != HB200_DT_FP32) {
      const int rc = try_ring<SRC_DT, MODE>(a, l);
      if (rc <= 0) return rc;
    }
    if (groups <= 4096) {
      if (vpt == 1) return launch_row<SRC_DT, 1, MODE, TIER>(a, l, threads);
      if (vpt == 2) return launch_row<SRC_DT, 2, MODE, TIER>(a, l, threads);
      return launch_row<SRC_DT, 4, MODE, TIER>(a, l, threads);
    }
  }
  return launch_row<SRC_DT, 0, MODE, TIER>(a, l, threads);
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
int launch_row_tier(const RowQuantArgs& a, const RowQuantLaunch& l) {
  constexpr int elem = sizeof(typename Src<SRC_DT>::T);
  switch (pick_tier(a, MODE, elem, a.weight_fp32 ? 4 : elem)) {
    case ROW_ALIGNED:
      return launch_row_size<SRC_DT, MODE, ROW_ALIGNED>(a, l);
    case ROW_PHASED:
      return launch_row_size<SRC_DT, MODE, ROW_PHASED>(a, l);
    default:
      return launch_row_size<SRC_DT, MODE, ROW_SCALAR>(a, l);
  }
}

template <int SRC_DT>
int launch_row_mode(const RowQuantArgs& a, const RowQuantLaunch& l) {
  if (a.weight == nullptr) return launch_row_tier<SRC_DT, 0>(a, l);
  return a.residual == nullptr ? launch_row_tier<SRC_DT, 1>(a, l) : launch_row_tier<SRC_DT, 2>(a, l);
}

}  // namespace

int launch_row_quantize(const RowQuantCall& c, DeviceCtx* ctx, int device, cudaStream_t stream) {
  const RowQuantLaunch l{c.M, ctx, device, stream};
  RowQuantArgs a;
  a.x = c.x;
  a.residual = c.residual;
  a.weight = c.weight;
  a.codes = c.codes;
  a.scales = c.scales;
  a.residual_out = c.residual_out;
  a.M = c.M;
  a.N = c.N;
  a.x_rs = c.x_rs;
  a.residual_rs = c.residual_rs;
  a.codes_rs = c.codes_rs;
  a.residual_out_rs = c.residual_out_rs;
  a.inv_n = 1.0f / static_cast<float>(c.N);
  a.eps = c.eps;
  a.weight_fp32 = c.weight_dtype == HB200_DT_FP32;
  a.weight_vectors = reinterpret_cast<uintptr_t>(c.weight) % 16 == 0;
  a.in_place = c.residual_out != nullptr && (c.residual_out == c.x || c.residual_out == c.residual);
  a.int8 = c.out_dtype == HB200_DT_INT8;
  switch (c.src_dtype) {
    case HB200_DT_FP16:
      return launch_row_mode<HB200_DT_FP16>(a, l);
    case HB200_DT_BF16:
      return launch_row_mode<HB200_DT_BF16>(a, l);
    default:
      return launch_row_mode<HB200_DT_FP32>(a, l);
  }
}

}  // namespace hb
