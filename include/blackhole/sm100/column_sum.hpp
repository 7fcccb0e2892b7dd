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

constexpr int kColumnSumCols = 128;       // columns per CTA of 1024 threads
using ColumnSumShared = float4[32][32];   // [row lane][4 columns]

// dst[col] = sum of src[i * stride + col] over i < count for the CTA's 128 columns: each warp takes
// every 32nd row, four columns per lane and eight rows in flight (one column per lane took four
// times the CTAs and 2 us more for five vectors of 148 x 8192), then the warps' sums are added in
// order.  `row0` (may be null) is one more row, added first.
__device__ __forceinline__ void column_sum_cta(const float* row0, const float* src, int64_t count,
                                               int64_t stride, float* dst, int cols, int col_block,
                                               ColumnSumShared& smem) {
  const int lane = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int col = col_block * kColumnSumCols + 4 * lane;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& v) {
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  };
  if (col < cols) {
    if (row0 && ry == 0) s = *reinterpret_cast<const float4*>(row0 + col);
    for (int64_t i = ry; i < count; i += 8 * 32) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = i + 32 * k < count ? *reinterpret_cast<const float4*>(src + (i + 32 * k) * stride + col)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) add(v[k]);
    }
  }
  smem[ry][lane] = s;
  __syncthreads();
  if (ry == 0 && col < cols) {
#pragma unroll 8
    for (int k = 1; k < 32; ++k) add(smem[k][lane]);
    *reinterpret_cast<float4*>(dst + col) = s;
  }
}

}  // namespace detail

#endif  // __CUDACC__

}  // namespace blackhole::sm100
