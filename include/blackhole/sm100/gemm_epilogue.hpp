#pragma once

// =====================================================================================
// blackhole / sm100 / epilogue of the block-scaled products and its gradient
// -------------------------------------------------------------------------------------
//     z = alpha * A . B^T + bias                       (FP32)
//     u = act(z), or gated: u[:, j] = act(z[:, 2j]) * z[:, 2j + 1]
//     D = bf16(u + beta * residual);   optionally Z = bf16(z), kept for the backward pass
//
// applied to the accumulators between TMEM and the store, in FP32, rounded once.  Gate and up
// features alternate (rows 2j and 2j + 1 of B), so a pair meets in one thread (one-SM and two-SM
// schedules: a thread owns a row's columns) or in two neighbouring lanes (skinny schedule).
//
// Backward, from the stored Z:  dZ = dD * act'(Z), gated dZ[:, 2j] = dD act'(g) u and
// dZ[:, 2j + 1] = dD act(g);  dbias = sum of its rows.  Bound by its bytes.
// =====================================================================================

#include <cmath>
#include <cstdint>

#include <cuda_runtime_api.h>

#include <blackhole/sm100/column_sum.hpp>
#include <blackhole/sm100/nvfp4_gemm_common.hpp>
#include <blackhole_sm100.h>

namespace blackhole::sm100 {

enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

namespace detail {

// Whether two byte ranges meet.
inline bool ranges_overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  if (!a || !b || an <= 0 || bn <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(bn) && y < x + static_cast<uintptr_t>(an);
}

}  // namespace detail

// Host-only check of an epilogue for an M x N product (after nvfp4_check_args).
inline cudaError_t epilogue_check_args(int M, int N, const void* D,
                                       const blackhole_sm100_epilogue* e) {
  if (!e) return cudaErrorInvalidValue;
  if (e->activation < kActNone || e->activation > kActSilu) return cudaErrorInvalidValue;
  if (e->gated && N % 16 != 0) return cudaErrorInvalidValue;   // D's rows stay 16-byte aligned
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (mis(e->bias) || mis(e->residual) || mis(e->Z)) return cudaErrorInvalidValue;
  if (e->residual && !std::isfinite(e->beta)) return cudaErrorInvalidValue;
  const int64_t d = int64_t(M) * (e->gated ? N / 2 : N) * 2, z = int64_t(M) * N * 2;
  if (e->residual && e->residual != D && detail::ranges_overlap(e->residual, d, D, d))
    return cudaErrorInvalidValue;
  if (detail::ranges_overlap(e->Z, z, D, d) || detail::ranges_overlap(e->Z, z, e->residual, d))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

#if defined(__CUDACC__)

namespace detail {

// ---- activations --------------------------------------------------------------------------
// exp and the divisions below are the fast forms (relative error a few 2^-23, against the 2^-9 of
// the BF16 result); every form keeps its relative accuracy in the tails, where 1 + tanh or 1 + erf
// would cancel.  |z| past 30 saturates the tanh form exactly in FP32, so its cubic is evaluated at
// the clamped z and cannot overflow.
__device__ __forceinline__ float act_sigmoid(float t) { return __fdividef(1.f, 1.f + __expf(-t)); }
__device__ __forceinline__ float gelu_tanh_arg(float z) {   // 2 sqrt(2 / pi) (z + 0.044715 z^3)
  const float c = fminf(fmaxf(z, -30.f), 30.f);
  return c * fmaf(0.0713548162726f, c * c, 1.59576912160573f);
}

template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (kAct == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (kAct == kActGelu) return 0.5f * z * erfcf(-0.707106781186548f * z);
  if constexpr (kAct == kActGeluTanh) return z * act_sigmoid(gelu_tanh_arg(z));
  if constexpr (kAct == kActSilu) return z * act_sigmoid(z);
  return z;
}

// act(z) and act'(z)
template <int kAct>
__device__ __forceinline__ void act_value_slope(float z, float& value, float& slope) {
  if constexpr (kAct == kActRelu) {
    value = act_value<kActRelu>(z);
    slope = z > 0.f ? 1.f : 0.f;
  } else if constexpr (kAct == kActGelu) {
    const float phi = 0.5f * erfcf(-0.707106781186548f * z);
    value = z * phi;
    slope = fmaf(z * 0.398942280401433f, __expf(-0.5f * z * z), phi);
  } else if constexpr (kAct == kActGeluTanh) {
    const float c = fminf(fmaxf(z, -30.f), 30.f);
    const float s = act_sigmoid(gelu_tanh_arg(z));
    value = z * s;
    slope = fmaf(c * s * (1.f - s), fmaf(0.214064448817800f, c * c, 1.59576912160573f), s);
  } else if constexpr (kAct == kActSilu) {
    const float s = act_sigmoid(z);
    value = z * s;
    slope = s * fmaf(z, 1.f - s, 1.f);
  } else {
    value = z;
    slope = 1.f;
  }
}

// Runs f with the activation as a compile-time constant.
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}

// ---- forward, on accumulators in registers --------------------------------------------------
struct EpilogueParams {
  CUtensorMap tmap_z;        // Z as D's map (one-SM and two-SM schedules, has_z only)
  const void* bias;
  const uint16_t* residual;  // BF16, rows of n_out
  uint16_t* z;               // BF16, rows of N (skinny schedule)
  float beta;
  int activation, gated, bias_bf16, has_z;
  int n_out;                 // columns of D
};

__device__ __forceinline__ float bf16_value(uint16_t bits) {
  return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}
__device__ __forceinline__ float epilogue_bias(const EpilogueParams& e, int n) {
  if (!e.bias) return 0.f;
  return e.bias_bf16 ? bf16_value(__ldg(static_cast<const uint16_t*>(e.bias) + n))
                     : __ldg(static_cast<const float*>(e.bias) + n);
}

// z of 32 consecutive columns of a row, in place of the accumulators' bits.
__device__ __forceinline__ void epilogue_z32(uint32_t (&v)[32], float alpha, const EpilogueParams& e,
                                             int col, int N) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(alpha * __uint_as_float(v[i]));
  if (!e.bias) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (col + 8 * g >= N) break;
    float b[8];
    if (e.bias_bf16) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.bias) + col + 8 * g));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[2 * i] = __uint_as_float(w[i] << 16);
        b[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    } else {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(e.bias) + col + 8 * g);
      const float4 lo = __ldg(q), hi = __ldg(q + 1);
      b[0] = lo.x; b[1] = lo.y; b[2] = lo.z; b[3] = lo.w;
      b[4] = hi.x; b[5] = hi.y; b[6] = hi.z; b[7] = hi.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * g + i] = __float_as_uint(__uint_as_float(v[8 * g + i]) + b[i]);
  }
}

// u of those columns: 32 values, or 16 (in v[0..15]) when gated.
__device__ __forceinline__ void epilogue_act32(uint32_t (&v)[32], const EpilogueParams& e) {
  with_activation(e.activation, [&](auto act) {
    constexpr int A = decltype(act)::value;
    if (e.gated) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = __float_as_uint(act_value<A>(__uint_as_float(v[2 * i])) * __uint_as_float(v[2 * i + 1]));
    } else if constexpr (A != kActNone) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(act_value<A>(__uint_as_float(v[i])));
    }
  });
}

// Adds beta * residual to 8 consecutive columns of D's row (col, row inside D).
__device__ __forceinline__ void epilogue_residual8(float (&f)[8], const EpilogueParams& e, int row, int col,
                                                   int M) {
  if (!e.residual || row >= M || col >= e.n_out) return;
  const uint4 q = *reinterpret_cast<const uint4*>(e.residual + int64_t(row) * e.n_out + col);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = fmaf(e.beta, __uint_as_float(w[i] << 16), f[2 * i]);
    f[2 * i + 1] = fmaf(e.beta, __uint_as_float(w[i] & 0xFFFF0000u), f[2 * i + 1]);
  }
}

// Fills the kernels' parameters; box_cols: columns of the schedule's store box (0: no map).
inline cudaError_t make_epilogue(EpilogueParams* p, const blackhole_sm100_epilogue& e, int M, int N,
                                 int box_cols) {
  p->bias = e.bias;
  p->residual = static_cast<const uint16_t*>(e.residual);
  p->z = static_cast<uint16_t*>(e.Z);
  p->beta = e.beta;
  p->activation = e.activation;
  p->gated = e.gated != 0;
  p->bias_bf16 = e.bias_is_bf16 != 0;
  p->has_z = e.Z != nullptr;
  p->n_out = e.gated ? N / 2 : N;
  if (e.Z && box_cols > 0) return make_d_tmap(&p->tmap_z, e.Z, M, N, box_cols);
  return cudaSuccess;
}

// ---- backward --------------------------------------------------------------------------------
constexpr int kEpilogueBackCols = 256;      // columns of Z per CTA: 32 lanes x 8

struct EpilogueBackwardParams {
  const uint16_t *d, *z;
  uint16_t* dz;
  float* dbias;
  float* ws;               // [row chunks][N] partial column sums
  int M, N, gated, chunks, rows_per_chunk;
};

template <int kAct>
__global__ void __launch_bounds__(256) epilogue_backward_kernel(const __grid_constant__ EpilogueBackwardParams p) {
  __shared__ float acc_s[8][kEpilogueBackCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * kEpilogueBackCols + lane * 8;
  const int row0 = blockIdx.y * p.rows_per_chunk;
  const int row1 = min(p.M, row0 + p.rows_per_chunk);
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (col < p.N) {
    for (int row = row0 + warp; row < row1; row += 8) {
      const int64_t at = int64_t(row) * p.N + col;
      const uint4 zq = *reinterpret_cast<const uint4*>(p.z + at);
      const uint32_t zw[4] = {zq.x, zq.y, zq.z, zq.w};
      float z[8], g[8], d[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[2 * i] = __uint_as_float(zw[i] << 16);
        z[2 * i + 1] = __uint_as_float(zw[i] & 0xFFFF0000u);
      }
      if (p.gated) {
        const uint2 q = *reinterpret_cast<const uint2*>(p.d + at / 2);
        const uint32_t w[2] = {q.x, q.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          d[2 * i] = __uint_as_float(w[i] << 16);
          d[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float value, slope;
          act_value_slope<kAct>(z[2 * i], value, slope);
          g[2 * i] = d[i] * z[2 * i + 1] * slope;
          g[2 * i + 1] = d[i] * value;
        }
      } else {
        const uint4 q = *reinterpret_cast<const uint4*>(p.d + at);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[2 * i] = __uint_as_float(w[i] << 16);
          d[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float value, slope;
          act_value_slope<kAct>(z[i], value, slope);
          g[i] = d[i] * slope;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += g[i];
      *reinterpret_cast<uint4*>(p.dz + at) = make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]),
                                                        pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7]));
    }
  }
  if (!p.dbias) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc_s[warp][lane * 8 + i] = acc[i];
  __syncthreads();
  const int c = blockIdx.x * kEpilogueBackCols + threadIdx.x;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += acc_s[w][threadIdx.x];
  if (c < p.N) (p.chunks == 1 ? p.dbias : p.ws + int64_t(blockIdx.y) * p.N)[c] = s;
}

static __global__ void __launch_bounds__(1024)
    epilogue_bias_sum_kernel(const __grid_constant__ EpilogueBackwardParams p) {
  __shared__ float smem[32 * 33];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  column_sum_cta(nullptr, p.ws, p.chunks, p.N, p.dbias, p.N, blockIdx.x, smem);
}

}  // namespace detail

#endif  // __CUDACC__

// Row chunks of the backward kernel: about eight CTAs per SM (148 SMs), each of whole sets of 8
// rows.  Fixed by the sizes, so the workspace and the order of the sums are too.
inline void epilogue_backward_chunks(int M, int N, int* chunks, int* rows_per_chunk) {
  const int64_t cols = (int64_t(N) + 255) / 256;
  int64_t want = (148 * 8 + cols - 1) / cols;
  if (want < 1) want = 1;
  int64_t rows = (int64_t(M) + want - 1) / want;
  rows = (rows + 7) / 8 * 8;
  *rows_per_chunk = static_cast<int>(rows);
  *chunks = static_cast<int>((M + rows - 1) / rows);
}

inline int64_t gemm_fused_backward_workspace_bytes(int M, int N) {
  if (M < 1 || N < 8 || N % 8 != 0) return -1;
  int chunks, rows;
  epilogue_backward_chunks(M, N, &chunks, &rows);
  return chunks == 1 ? 0 : int64_t(chunks) * N * 4;
}

// Host-only check.
inline cudaError_t gemm_fused_backward_check(int M, int N, const void* dD, const void* Z, const void* dZ,
                                             const float* dbias, int activation, int gated,
                                             const void* workspace, int64_t workspace_bytes) {
  if (M < 1 || N < 8 || N % 8 != 0 || (gated && N % 16 != 0)) return cudaErrorInvalidValue;
  if (activation < kActNone || activation > kActSilu) return cudaErrorInvalidValue;
  if (!dD || !Z || !dZ) return cudaErrorInvalidValue;
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (mis(dD) || mis(Z) || mis(dZ) || mis(dbias) || mis(workspace)) return cudaErrorInvalidValue;
  if (int64_t(M) * N > (int64_t(1) << 46)) return cudaErrorInvalidValue;
  const int64_t z = int64_t(M) * N * 2, d = gated ? z / 2 : z;
  if (dZ != Z && detail::ranges_overlap(dZ, z, Z, z)) return cudaErrorInvalidValue;
  if ((dZ != dD || gated) && detail::ranges_overlap(dZ, z, dD, d)) return cudaErrorInvalidValue;
  const int64_t need = gemm_fused_backward_workspace_bytes(M, N);
  if (dbias && need > 0 && (!workspace || workspace_bytes < need)) return cudaErrorInvalidValue;
  return cudaSuccess;
}

#if defined(__CUDACC__)

inline cudaError_t gemm_fused_backward(int M, int N, const void* dD, const void* Z, void* dZ, float* dbias,
                                       int activation, int gated, void* workspace,
                                       int64_t workspace_bytes, cudaStream_t stream) {
  cudaError_t e = gemm_fused_backward_check(M, N, dD, Z, dZ, dbias, activation, gated, workspace,
                                            workspace_bytes);
  if (e != cudaSuccess) return e;
  detail::EpilogueBackwardParams p;
  p.d = static_cast<const uint16_t*>(dD);
  p.z = static_cast<const uint16_t*>(Z);
  p.dz = static_cast<uint16_t*>(dZ);
  p.dbias = dbias;
  p.ws = static_cast<float*>(workspace);
  p.M = M;
  p.N = N;
  p.gated = gated != 0;
  epilogue_backward_chunks(M, N, &p.chunks, &p.rows_per_chunk);
  const dim3 grid((N + detail::kEpilogueBackCols - 1) / detail::kEpilogueBackCols, p.chunks);
  void (*kernel)(detail::EpilogueBackwardParams) = nullptr;
  switch (activation) {
    case kActRelu: kernel = detail::epilogue_backward_kernel<kActRelu>; break;
    case kActGelu: kernel = detail::epilogue_backward_kernel<kActGelu>; break;
    case kActGeluTanh: kernel = detail::epilogue_backward_kernel<kActGeluTanh>; break;
    case kActSilu: kernel = detail::epilogue_backward_kernel<kActSilu>; break;
    default: kernel = detail::epilogue_backward_kernel<kActNone>; break;
  }
  e = detail::launch_pdl(kernel, grid, dim3(256), 0, stream, p);
  if (e != cudaSuccess) return e;
  if (dbias && p.chunks > 1) {
    e = detail::launch_pdl(detail::epilogue_bias_sum_kernel, dim3((N + 31) / 32), dim3(1024), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

#endif  // __CUDACC__

}  // namespace blackhole::sm100
