#pragma once

// Second stage of a column sum over many rows: the first stage (a kernel whose CTAs each walk a
// range of rows) leaves one FP32 partial row per CTA, and this kernel adds those in a fixed
// order, so results do not depend on timing.  A job is one output vector: `count` partial rows
// of `cols` values, `stride` floats apart.

#include <cstdint>

#include <cuda_runtime_api.h>

#include <blackhole/sm100/nvfp4_gemm_common.hpp>

namespace blackhole::sm100 {

#if defined(__CUDACC__)

namespace detail {

// Sum of src[i * stride + col] for i = first, first + 32, ... < count on a warp's lane, then over
// the CTA's warps: 1024 threads as 32 columns x 32 row lanes.  `row0` (may be null) is one more
// partial row added first.
__device__ __forceinline__ void column_sum_cta(const float* row0, const float* src, int64_t count,
                                               int64_t stride, float* dst, int cols, int col_block,
                                               float* smem) {
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int col = col_block * 32 + cx;
  float s = 0.f;
  if (col < cols) {
    if (row0 && ry == 0) s = row0[col];
    int64_t i = ry;
    for (; i + 7 * 32 < count; i += 8 * 32) {       // eight loads in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = src[(i + 32 * k) * stride + col];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < count ? src[(i + 32 * k) * stride + col] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k];
  }
  smem[ry * 33 + cx] = s;
  __syncthreads();
  // warp ry now owns column ry: one value per lane
  float t = smem[cx * 33 + ry];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  const int out = col_block * 32 + ry;
  if (cx == 0 && out < cols) dst[out] = t;
}

}  // namespace detail

#endif  // __CUDACC__

}  // namespace blackhole::sm100
