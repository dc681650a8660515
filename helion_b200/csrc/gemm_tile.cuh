// Tile order and output staging shared by the persistent GEMM kernels (fp8_gemm.cu, gated_gemm.cuh).
#pragma once

#include "common.cuh"
#include "host.h"

namespace hb {

struct TileCoord {
  int m_blk;
  int n_blk;
};

// Grouped ("L2 swizzled") order: consecutive tile indices walk down GROUP_M row blocks before
// moving to the next column block, so CTAs that run at the same time share x and y tiles in L2.
__device__ __forceinline__ TileCoord tile_coord(int tile, int m_tiles, int n_tiles, int group_m) {
  const int per_group = group_m * n_tiles;
  const int group = tile / per_group;
  const int first_m = group * group_m;
  const int rows = min(m_tiles - first_m, group_m);
  const int in_group = tile - group * per_group;
  TileCoord c;
  c.m_blk = first_m + in_group % rows;
  c.n_blk = in_group / rows;
  return c;
}

// Epilogue through shared memory and TMA: one warp stages a 32-row x 32-column block of converted
// outputs (row = lane) in a swizzled buffer and one lane stores it with a tiled bulk copy, which
// writes full row segments (instead of 32 scattered 16-byte pieces per store instruction) and clips
// rows beyond M / columns beyond N.  `stage` holds NBUF buffers of 32 x ROW_BYTES; the store that last
// used a buffer is waited for (its smem reads only) before the buffer is rewritten: all groups but the latest KEEP
// (a caller that takes turns with other buffers of its own passes how many stores lie between two uses of this one).
template <int OUT_DT>
struct StagedStore {
  static constexpr bool OUT32 = OUT_DT == HB200_DT_FP32;
  static constexpr int ROW_BYTES = OUT32 ? 128 : 64;
  static constexpr int STG_BYTES = 32 * ROW_BYTES;
  static constexpr int NBUF = OUT32 ? 1 : 2;  // 4 KB per warp either way

  // `layer` (with SLICED maps): which of the matrices of a three-dimensional output map the block goes to.
  template <int KEEP = NBUF - 1, bool SLICED = false>
  __device__ static __forceinline__ void store(const uint32_t (&r)[32], uint8_t* stage, uint32_t chunk_count, int lane,
                                               const CUtensorMap* tmap_out, int col, int row0, bool inside,
                                               unsigned long long* trace = nullptr, int layer = 0) {
    uint8_t* buf = stage + (chunk_count % NBUF) * STG_BYTES;
    if (lane == 0) tma_store_wait_read<KEEP>();
    __syncwarp();
#ifdef HB_GEMM_TRACE
    if (trace != nullptr) asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(trace[0]));
#endif
    // 16-byte chunk j of row r lives at chunk j ^ ((r >> 1) & 3) (64-byte rows, SWIZZLE_64B) or
    // j ^ (r & 7) (128-byte rows, SWIZZLE_128B): the pattern the output tensor map expects
    const uint32_t swz = OUT32 ? static_cast<uint32_t>(lane & 7) : static_cast<uint32_t>((lane >> 1) & 3);
    uint8_t* dst_row = buf + lane * ROW_BYTES;
    if constexpr (OUT32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        *reinterpret_cast<uint4*>(dst_row + ((static_cast<uint32_t>(j) ^ swz) << 4)) =
            make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t p[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float lo = __uint_as_float(r[8 * j + 2 * q]);
          const float hi = __uint_as_float(r[8 * j + 2 * q + 1]);
          p[q] = (OUT_DT == HB200_DT_BF16) ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
        }
        *reinterpret_cast<uint4*>(dst_row + ((static_cast<uint32_t>(j) ^ swz) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      // blocks that lie wholly outside the matrix are not stored at all (partial ones are clipped)
      if (inside) {
        if constexpr (SLICED) tma_store_3d(tmap_out, buf, col, row0, layer);
        else tma_store_2d(tmap_out, buf, col, row0);
      }
      tma_store_commit();
    }
  }
};

}  // namespace hb
