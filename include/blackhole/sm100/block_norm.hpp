#pragma once

// =====================================================================================
// blackhole / sm100 / norms before and after a block, fused with its gate and residual scale
// -------------------------------------------------------------------------------------
// Between two block-scaled products of a transformer stands, per row of H features,
//
//     p = o                       or  norm_post(o)       (o: the block's BF16 result)
//     h = x + scale * g * p                              (x: residual stream, g: gate)
//     y = norm(h) * weight + bias                        (the next block's input)
//
// with norm either RMS (v / sqrt(mean(v^2) + eps)) or layer ((v - mean) / sqrt(var + eps)).
// One kernel reads x and o once and writes h and y once; y leaves as BF16, FP32 or quantised as
// the next product's A operand (the recipes of nvfp4_quant.hpp on the FP32 y, no BF16 step in
// between), scale factors in the 128x4 layout.  Everything between the loads and the stores is
// FP32; y uses the FP32 h, not its stored rounding.
//
// Backward (a = dy * weight, n = (h - mean) * rstd from the stored h and statistics):
//     dh' = dh + rstd * (a - [mean(a)] - n * mean(a * n));   dx = dh'
//     dp  = scale * g * dh';   dg = scale * dh' * p, summed over the rows that share a gate row
//     do  = dp, or norm_post's gradient of it (same form)
//     dweight = sum dy * n, dbias = sum dy, and the same two of the post norm
// ([...]: layer norm only).
//
// A row is worked on by one CTA (H <= 8192) or a cluster of two (H <= 16384), 16 columns per
// thread as two 8-column vectors.
// =====================================================================================

#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cuda_runtime_api.h>

#include <blackhole/common/sf_layout.hpp>
#include <blackhole/sm100/column_sum.hpp>
#include <blackhole/sm100/gemm_epilogue.hpp>
#include <blackhole/sm100/nvfp4_gemm_common.hpp>
#include <blackhole/sm100/nvfp4_quant.hpp>
#include <blackhole_sm100.h>

namespace blackhole::sm100 {

constexpr int kNormMaxH = 16384;
constexpr int kNormSliceH = 8192;     // columns one CTA works on: 512 threads x 16

enum NormOut : int { kOutBf16 = 0, kOutF32 = 1, kOutNvfp4 = 2, kOutMxfp4 = 3, kOutMxfp8 = 4 };

namespace norm_detail {

struct Geometry {
  int cluster;      // CTAs per row: 1 or 2
  int slice;        // columns of a row per CTA (a multiple of 128 when cluster == 2)
  int threads;      // threads per CTA, 16 columns each
};
inline Geometry geometry(int H) {
  Geometry g;
  g.cluster = H > kNormSliceH ? 2 : 1;
  g.slice = g.cluster == 1 ? H : (((H + 1) / 2 + 127) / 128 * 128);
  g.threads = ((g.slice + 15) / 16 + 31) / 32 * 32;
  return g;
}

// Row ranges of the backward kernel: `teams` CTAs (or clusters) of `rows_per_team` consecutive
// rows.  Fixed by the sizes alone (148 SMs, 512 resident threads on each), so the workspace size
// and the order of the column sums do not depend on the device's state.
struct Teams {
  int teams;
  int rows_per_team;
};
inline Teams backward_teams(int rows, int H) {
  const Geometry g = geometry(H);
  const int per_sm = std::max(1, 512 / g.threads);
  const int cap = std::max(1, 148 * per_sm / g.cluster);
  Teams t;
  t.rows_per_team = (rows + cap - 1) / cap;
  t.teams = (rows + t.rows_per_team - 1) / t.rows_per_team;
  return t;
}

}  // namespace norm_detail

inline int64_t block_norm_backward_workspace_bytes(int rows, int H, int has_gate, int gate_rows) {
  if (rows < 1 || H < 8 || H > kNormMaxH || H % 8 != 0 || gate_rows < 0) return -1;
  const int64_t teams = norm_detail::backward_teams(rows, H).teams;
  const int64_t vectors = 4 + ((has_gate && gate_rows != 1) ? 2 : 0);
  return teams * vectors * H * 4;
}

inline cudaError_t block_norm_check(const blackhole_sm100_block_norm_args& a) {
  if (a.rows < 1 || a.H < 8 || a.H > kNormMaxH || a.H % 8 != 0) return cudaErrorInvalidValue;
  if (a.kind < 0 || a.kind > 1 || a.gate_rows < 0) return cudaErrorInvalidValue;
  if (!(a.eps >= 0.0f) || !std::isfinite(a.eps) || !std::isfinite(a.scale))
    return cudaErrorInvalidValue;
  if (a.out_format < kOutBf16 || a.out_format > kOutMxfp8) return cudaErrorInvalidValue;
  if (!a.x || (!a.out && !a.h)) return cudaErrorInvalidValue;
  // without a block result there is nothing to gate, to norm or to add
  if (!a.o && (a.gate || a.post_norm || a.h)) return cudaErrorInvalidValue;
  if (!a.post_norm && (a.post_weight || a.post_bias)) return cudaErrorInvalidValue;
  if (!a.out && (a.weight || a.bias || a.sf)) return cudaErrorInvalidValue;
  const bool quant = a.out && a.out_format >= kOutNvfp4;
  if (quant != (a.sf != nullptr)) return cudaErrorInvalidValue;
  if (quant && a.H % (a.out_format == kOutNvfp4 ? 16 : 32) != 0) return cudaErrorInvalidValue;
  if (quant && a.out_format == kOutNvfp4 && (!(a.global_scale > 0.0f) || !std::isfinite(a.global_scale)))
    return cudaErrorInvalidValue;
  const void* ptrs[] = {a.x, a.o, a.gate, a.weight, a.bias, a.post_weight, a.post_bias,
                        a.h, a.out, a.sf, a.stats};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorInvalidValue;
  const int64_t n = int64_t(a.rows) * a.H;
  const int64_t xb = n * (a.x_is_bf16 ? 2 : 4);
  const int64_t yb = a.out_format == kOutBf16 ? n * 2 : a.out_format == kOutF32 ? n * 4
                     : a.out_format == kOutMxfp8 ? n : n / 2;
  if (a.h && a.h != a.x && detail::ranges_overlap(a.h, xb, a.x, xb)) return cudaErrorInvalidValue;
  if (detail::ranges_overlap(a.h, xb, a.o, n * 2) || detail::ranges_overlap(a.h, xb, a.out, yb) ||
      detail::ranges_overlap(a.out, yb, a.x, xb) || detail::ranges_overlap(a.out, yb, a.o, n * 2))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

inline cudaError_t block_norm_backward_check(const blackhole_sm100_block_norm_backward_args& a) {
  if (a.rows < 1 || a.H < 8 || a.H > kNormMaxH || a.H % 8 != 0) return cudaErrorInvalidValue;
  if (a.kind < 0 || a.kind > 1 || a.gate_rows < 0 || !std::isfinite(a.scale))
    return cudaErrorInvalidValue;
  if (!a.h || !a.stats || !a.dx || (!a.dy && !a.dh)) return cudaErrorInvalidValue;
  if (!a.o && (a.gate || a.post_norm || a.d_o || a.dgate)) return cudaErrorInvalidValue;
  if (a.o && !a.d_o) return cudaErrorInvalidValue;
  if (!a.post_norm && (a.post_weight || a.post_bias || a.dpost_weight || a.dpost_bias))
    return cudaErrorInvalidValue;
  if (!a.gate && a.dgate) return cudaErrorInvalidValue;
  const void* ptrs[] = {a.h, a.stats, a.dy, a.dh, a.o, a.gate, a.weight, a.post_weight,
                        a.post_bias, a.dx, a.d_o, a.dweight, a.dbias, a.dpost_weight,
                        a.dpost_bias, a.dgate, a.workspace};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorInvalidValue;
  const bool sums = a.dweight || a.dbias || a.dpost_weight || a.dpost_bias ||
                    (a.dgate && a.gate_rows != 1);
  if (sums) {
    const int64_t need = block_norm_backward_workspace_bytes(a.rows, a.H, a.gate != nullptr, a.gate_rows);
    if (!a.workspace || a.workspace_bytes < need) return cudaErrorInvalidValue;
  }
  const int64_t n = int64_t(a.rows) * a.H;
  const int64_t xb = n * (a.x_is_bf16 ? 2 : 4);
  if (a.dx != a.dh && detail::ranges_overlap(a.dx, xb, a.dh, xb)) return cudaErrorInvalidValue;
  if (detail::ranges_overlap(a.dx, xb, a.h, xb) || detail::ranges_overlap(a.dx, xb, a.dy, n * 2) ||
      detail::ranges_overlap(a.dx, xb, a.o, n * 2) || detail::ranges_overlap(a.dx, xb, a.d_o, n * 2) ||
      detail::ranges_overlap(a.d_o, n * 2, a.h, xb) || detail::ranges_overlap(a.d_o, n * 2, a.dh, xb) ||
      detail::ranges_overlap(a.d_o, n * 2, a.dy, n * 2) || detail::ranges_overlap(a.d_o, n * 2, a.o, n * 2))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

#if defined(__CUDACC__)

namespace norm_detail {

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// A vector of parameters or gates, BF16 or FP32 (uniform over the launch).
__device__ __forceinline__ void load8_any(const void* p, int64_t at, int is_bf16, float (&v)[8]) {
  if (is_bf16) load8(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load8(static_cast<const float*>(p) + at, v);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(detail::pack_bf16x2(v[0], v[1]), detail::pack_bf16x2(v[2], v[3]),
                 detail::pack_bf16x2(v[4], v[5]), detail::pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sums over the threads of a row's CTA or cluster, the same value in every thread, added in a
// fixed order.  Two slot sets in turn: a set is written again only after a later barrier that
// every reader of it has passed.
template <int kCl, int kN>
struct RowSum {
  float (*slots)[kN][kCl * 16];   // [2][kN][CTA * 16 + warp], zeroed before first use
  int set = 0;

  __device__ __forceinline__ void operator()(float (&v)[kN]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] = warp_sum(v[k]);
    if (kCl == 1 && blockDim.x == 32) return;
    if constexpr (kCl == 1) {
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < kN; ++k) slots[set][k][warp] = v[k];
      __syncthreads();
    } else {
      const int rank = static_cast<int>(ptx::cluster_ctarank());
      if (lane < kCl)
#pragma unroll
        for (int k = 0; k < kN; ++k) {
          const uint32_t a = ptx::mapa_shared(
              ptx::smem_u32(&slots[set][k][rank * 16 + warp]), static_cast<uint32_t>(lane));
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v[k]) : "memory");
        }
      ptx::cluster_sync();
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      float s = 0.f;
      const float4* q = reinterpret_cast<const float4*>(slots[set][k]);
#pragma unroll
      for (int i = 0; i < kCl * 4; ++i) {
        const float4 t = q[i];
        s += (t.x + t.y) + (t.z + t.w);
      }
      v[k] = s;
    }
    set ^= 1;
  }
};

struct NormParams {
  const void *x, *o, *gate, *weight, *bias, *post_weight, *post_bias;
  void *h, *out;
  uint8_t* sf;
  float* stats;
  int rows, H, slice, teams;
  int gate_rows, param_bf16, gate_bf16, out_format;
  float scale, eps, global_scale;
};

// Quantises 8 consecutive columns of this thread's row; neighbouring lanes hold the other
// columns of the 16- or 32-column block.  Every lane of the warp calls it (`live` false: past
// the row's end, all zero).  Recipes and roundings are those of nvfp4_quant.hpp.
template <class Store32, class Store64>
__device__ __forceinline__ uint32_t quantize8(const float (&y)[8], bool live, int fmt, float g,
                                              Store32 store32, Store64 store64) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(y[i]));
  m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  uint32_t code = 0;
  if (fmt == kOutNvfp4) {
    uint32_t q = 0;
    if (live && m > 0.f) {
      code = quant_detail::ue4m3_cvt((m / 6.0f) / g);
      const float s = quant_detail::ue4m3_value(code);
      if (s != 0.f) {
        const float scale = s * g;
        q = quant_detail::e2m1x4_cvt(y[0] / scale, y[1] / scale, y[2] / scale, y[3] / scale) |
            (quant_detail::e2m1x4_cvt(y[4] / scale, y[5] / scale, y[6] / scale, y[7] / scale) << 16);
      }
    }
    store32(q);
    return code;
  }
  m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  const int ebits = static_cast<int>((__float_as_uint(m) >> 23) & 0xFFu);
  int e = ebits == 0 ? -127 : ebits - (fmt == kOutMxfp8 ? 135 : 129);
  e = max(-127, min(127, e));
  code = live ? static_cast<uint32_t>(e + 127) : 0u;
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  if (fmt == kOutMxfp4) {
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) q |= quant_detail::e2m1_rne(y[i] * inv) << (4 * i);
    store32(q);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = quant_detail::e4m3x2_satfinite(y[4 * i] * inv, y[4 * i + 1] * inv) |
             (quant_detail::e4m3x2_satfinite(y[4 * i + 2] * inv, y[4 * i + 3] * inv) << 16);
    store64(make_uint2(w[0], w[1]));
  }
  return code;
}

template <class TX, bool kLayer, bool kPost, int kCl>
__global__ void __cluster_dims__(kCl, 1, 1) __launch_bounds__(512)
    block_norm_kernel(const __grid_constant__ NormParams p) {
#if defined(BLACKHOLE_ARCH_SM100)
  __shared__ __align__(16) float slots[2][1][kCl * 16];
  const int rank = kCl == 1 ? 0 : static_cast<int>(ptx::cluster_ctarank());
  const int team = blockIdx.x / kCl;
  const int T = blockDim.x, tid = threadIdx.x, lane = tid & 31;
  const int H = p.H;
  const int c0 = rank * p.slice, c1 = min(H, c0 + p.slice);
  ptx::pdl_launch_dependents();
  for (int i = tid; i < 2 * kCl * 16; i += T) (&slots[0][0][0])[i] = 0.f;
  if constexpr (kCl == 1) __syncthreads();
  else ptx::cluster_sync();
  RowSum<kCl, 1> row_sum{slots};
  auto sum = [&](float v) {
    float a[1] = {v};
    row_sum(a);
    return a[0];
  };
  ptx::pdl_wait_prior_grid();

  int col[2];
  bool live[2];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    col[v] = c0 + (v * T + tid) * 8;
    live[v] = col[v] < c1;
  }
  const float inv_h = 1.0f / static_cast<float>(H);
  for (int row = team; row < p.rows; row += p.teams) {
    const int64_t at = int64_t(row) * H;
    float h[2][8], mean_post = 0.f, rstd_post = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[v][i] = 0.f;
      if (live[v]) load8(static_cast<const TX*>(p.x) + at + col[v], h[v]);
    }
    if (p.o) {
      float o[2][8];
#pragma unroll
      for (int v = 0; v < 2; ++v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[v][i] = 0.f;
        if (live[v]) load8(static_cast<const __nv_bfloat16*>(p.o) + at + col[v], o[v]);
      }
      if constexpr (kPost) {
        float s = 0.f;
        if constexpr (kLayer) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s += o[i / 8][i % 8];
          mean_post = sum(s) * inv_h;
        }
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float d = o[i / 8][i % 8] - mean_post;
          s += live[i / 8] ? d * d : 0.f;
        }
        rstd_post = __frsqrt_rn(sum(s) * inv_h + p.eps);
      }
      const int64_t gate_at = p.gate_rows ? int64_t(row / p.gate_rows) * H : 0;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (!live[v]) continue;
        if constexpr (kPost) {
#pragma unroll
          for (int i = 0; i < 8; ++i) o[v][i] = (o[v][i] - mean_post) * rstd_post;
          if (p.post_weight) {
            float w[8];
            load8_any(p.post_weight, col[v], p.param_bf16, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[v][i] *= w[i];
          }
          if (p.post_bias) {
            float w[8];
            load8_any(p.post_bias, col[v], p.param_bf16, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[v][i] += w[i];
          }
        }
        if (p.gate) {
          float w[8];
          load8_any(p.gate, gate_at + col[v], p.gate_bf16, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[v][i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[v][i] = fmaf(p.scale, o[v][i], h[v][i]);
        if (p.h) store8(static_cast<TX*>(p.h) + at + col[v], h[v]);
      }
    }
    if (!p.out && !p.stats) continue;
    float mean = 0.f, s = 0.f;
    if constexpr (kLayer) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s += h[i / 8][i % 8];
      mean = sum(s) * inv_h;
    }
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = h[i / 8][i % 8] - mean;
      s += live[i / 8] ? d * d : 0.f;
    }
    const float rstd = __frsqrt_rn(sum(s) * inv_h + p.eps);
    if (p.stats && rank == 0 && tid == 0)
      reinterpret_cast<float4*>(p.stats)[row] = make_float4(mean_post, rstd_post, mean, rstd);
    if (!p.out) continue;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = live[v] ? (h[v][i] - mean) * rstd : 0.f;
      if (live[v] && p.weight) {
        float w[8];
        load8_any(p.weight, col[v], p.param_bf16, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= w[i];
      }
      if (live[v] && p.bias) {
        float w[8];
        load8_any(p.bias, col[v], p.param_bf16, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += w[i];
      }
      if (p.out_format == kOutBf16) {
        if (live[v]) store8(static_cast<__nv_bfloat16*>(p.out) + at + col[v], y);
      } else if (p.out_format == kOutF32) {
        if (live[v]) store8(static_cast<float*>(p.out) + at + col[v], y);
      } else {
        uint8_t* const out = static_cast<uint8_t*>(p.out);
        const uint32_t code = quantize8(
            y, live[v], p.out_format, p.global_scale,
            [&](uint32_t q) {
              if (live[v]) *reinterpret_cast<uint32_t*>(out + (at + col[v]) / 2) = q;
            },
            [&](uint2 q) {
              if (live[v]) *reinterpret_cast<uint2*>(out + at + col[v]) = q;
            });
        // four groups' codes make one word of the row: 2 (NVFP4) or 4 lanes per group
        const int per = p.out_format == kOutNvfp4 ? 2 : 4;
        uint32_t word = code << (8 * ((lane / per) & 3));
        word = (lane % per) == 0 ? word : 0u;
        for (int o = 4 * per / 2; o > 0; o >>= 1) word |= __shfl_xor_sync(0xFFFFFFFFu, word, o);
        if ((lane & (4 * per - 1)) == 0 && col[v] < c1)
          *reinterpret_cast<uint32_t*>(
              p.sf + sf_offset_vs(row, col[v] / (8 * per), H, 8 * per)) = word;
      }
    }
  }
  // scale factors of the layout's padding rows
  if (p.out && p.sf && rank == 0) {
    const int vs = p.out_format == kOutNvfp4 ? 16 : 32;
    const int words = static_cast<int>(sf_k_atoms_vs(H, vs));
    const int pad = (p.rows + 127) / 128 * 128 - p.rows;
    for (int64_t i = int64_t(team) * T + tid; i < int64_t(pad) * words; i += int64_t(p.teams) * T)
      *reinterpret_cast<uint32_t*>(
          p.sf + sf_offset_vs(p.rows + int(i / words), 4 * (i % words), H, vs)) = 0u;
  }
  if constexpr (kCl > 1) ptx::cluster_sync();   // no CTA leaves while its partner writes its slots
#endif
}

struct NormBackwardParams {
  const void *h, *dy, *dh, *o, *gate, *weight, *post_weight, *post_bias;
  const float* stats;
  void *dx, *d_o;
  float *dweight, *dbias, *dpost_weight, *dpost_bias, *dgate;
  float* ws;            // [vector][team][H]: dweight, dbias, dpost_weight, dpost_bias, gate edges
  int rows, H, slice, teams, rows_per_team;
  int gate_rows, param_bf16, gate_bf16;
  float scale;
};

template <class TX, bool kLayer, bool kPost, bool kGate, int kCl>
__global__ void __cluster_dims__(kCl, 1, 1) __launch_bounds__(512, 1)
    block_norm_backward_kernel(const __grid_constant__ NormBackwardParams p) {
#if defined(BLACKHOLE_ARCH_SM100)
  __shared__ __align__(16) float slots[2][2][kCl * 16];
  const int rank = kCl == 1 ? 0 : static_cast<int>(ptx::cluster_ctarank());
  const int team = blockIdx.x / kCl;
  const int T = blockDim.x, tid = threadIdx.x;
  const int H = p.H;
  const int c0 = rank * p.slice, c1 = min(H, c0 + p.slice);
  ptx::pdl_launch_dependents();
  for (int i = tid; i < 4 * kCl * 16; i += T) (&slots[0][0][0])[i] = 0.f;
  if constexpr (kCl == 1) __syncthreads();
  else ptx::cluster_sync();
  RowSum<kCl, 2> row_sum{slots};
  ptx::pdl_wait_prior_grid();

  int col[2];
  bool live[2];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    col[v] = c0 + (v * T + tid) * 8;
    live[v] = col[v] < c1;
  }
  const float inv_h = 1.0f / static_cast<float>(H);
  const int row0 = team * p.rows_per_team, row1 = min(p.rows, row0 + p.rows_per_team);
  const int64_t vec = int64_t(p.teams) * H;           // floats of one vector's partials
  float dw[16], db[kLayer ? 16 : 1], dwp[kPost ? 16 : 1], dbp[kPost && kLayer ? 16 : 1],
      dg[kGate ? 16 : 1];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    dw[i] = 0.f;
    if constexpr (kLayer) db[i] = 0.f;
    if constexpr (kPost) dwp[i] = 0.f;
    if constexpr (kPost && kLayer) dbp[i] = 0.f;
    if constexpr (kGate) dg[i] = 0.f;
  }
  for (int row = row0; row < row1; ++row) {
    const int64_t at = int64_t(row) * H;
    const float4 st = reinterpret_cast<const float4*>(p.stats)[row];
    float d[2][8];                                    // dh', then dp
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[v][i] = 0.f;
      if (live[v] && p.dh) load8(static_cast<const TX*>(p.dh) + at + col[v], d[v]);
    }
    if (p.dy) {
      float n[2][8], a[2][8], s[2] = {0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 2; ++v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) n[v][i] = a[v][i] = 0.f;
        if (!live[v]) continue;
        load8(static_cast<const TX*>(p.h) + at + col[v], n[v]);
        load8(static_cast<const __nv_bfloat16*>(p.dy) + at + col[v], a[v]);
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
        if (p.weight) load8_any(p.weight, col[v], p.param_bf16, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[v][i] = (n[v][i] - st.z) * st.w;
          dw[8 * v + i] = fmaf(a[v][i], n[v][i], dw[8 * v + i]);
          if constexpr (kLayer) db[8 * v + i] += a[v][i];
          a[v][i] *= w[i];
          s[0] = fmaf(a[v][i], n[v][i], s[0]);
          if constexpr (kLayer) s[1] += a[v][i];
        }
      }
      row_sum(s);
      const float along = s[0] * inv_h, mean_a = s[1] * inv_h;
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (live[v])
            d[v][i] = fmaf(st.w, a[v][i] - (kLayer ? mean_a : 0.f) - n[v][i] * along, d[v][i]);
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (live[v]) store8(static_cast<TX*>(p.dx) + at + col[v], d[v]);
    if (!p.o) continue;

    const int group = (kGate && p.gate_rows) ? row / p.gate_rows : 0;
    float n[2][8], s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) n[v][i] = 0.f;
      if (!live[v]) continue;
      load8(static_cast<const __nv_bfloat16*>(p.o) + at + col[v], n[v]);
      float w[8];
      if constexpr (kPost) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[v][i] = (n[v][i] - st.x) * st.y;
          w[i] = 1.f;
        }
        if (p.post_weight) load8_any(p.post_weight, col[v], p.param_bf16, w);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) d[v][i] *= p.scale;
      if constexpr (kGate) {
        float pv[8], g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pv[i] = kPost ? n[v][i] * w[i] : n[v][i];
        if (kPost && p.post_bias) {
          float b[8];
          load8_any(p.post_bias, col[v], p.param_bf16, b);
#pragma unroll
          for (int i = 0; i < 8; ++i) pv[i] += b[i];
        }
        load8_any(p.gate, int64_t(group) * H + col[v], p.gate_bf16, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dg[8 * v + i] = fmaf(d[v][i], pv[i], dg[8 * v + i]);
          d[v][i] *= g[i];
        }
      }
      if constexpr (kPost) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dwp[8 * v + i] = fmaf(d[v][i], n[v][i], dwp[8 * v + i]);
          if constexpr (kLayer) dbp[8 * v + i] += d[v][i];
          d[v][i] *= w[i];
          s[0] = fmaf(d[v][i], n[v][i], s[0]);
          if constexpr (kLayer) s[1] += d[v][i];
        }
      }
    }
    if constexpr (kPost) {
      row_sum(s);
      const float along = s[0] * inv_h, mean_a = s[1] * inv_h;
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          d[v][i] = st.y * (d[v][i] - (kLayer ? mean_a : 0.f) - n[v][i] * along);
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (live[v]) store8(static_cast<__nv_bfloat16*>(p.d_o) + at + col[v], d[v]);

    if constexpr (kGate) {
      // last row of this gate row's group in this team: the sum is whole (stored), or an edge
      // piece for the second kernel: slot 0 if the group began in an earlier team, else slot 1
      const bool last = row + 1 == row1 || (p.gate_rows && (row + 1) % p.gate_rows == 0);
      if (last) {
        const int64_t g0 = int64_t(group) * p.gate_rows;
        const int64_t g1 = p.gate_rows ? min(int64_t(p.rows), g0 + p.gate_rows) : p.rows;
        if (p.dgate) {
          float* dst = g0 >= row0 && g1 <= row1 ? p.dgate + int64_t(group) * H
                                                : p.ws + (g0 < row0 ? 4 : 5) * vec + int64_t(team) * H;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = dg[8 * v + i];
            if (live[v]) store8(dst + col[v], t);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dg[i] = 0.f;
      }
    }
  }
  auto park = [&](const float* out, int which, const float* acc) {
    if (!out) return;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = acc[8 * v + i];
      if (live[v]) store8(p.ws + which * vec + int64_t(team) * H + col[v], t);
    }
  };
  park(p.dweight, 0, dw);
  if constexpr (kLayer) park(p.dbias, 1, db);
  if constexpr (kPost) park(p.dpost_weight, 2, dwp);
  if constexpr (kPost && kLayer) park(p.dpost_bias, 3, dbp);
  if constexpr (kCl > 1) ptx::cluster_sync();
#endif
}

// Adds the teams' partials: y = 0..3 the four parameter vectors, y = 3 + c (c = 1..teams-1) the
// gate group that crosses into team c, if c is the first team it crosses into.
static __global__ void __launch_bounds__(1024)
    block_norm_sums_kernel(const __grid_constant__ NormBackwardParams p) {
  __shared__ float smem[32 * 33];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  const int64_t vec = int64_t(p.teams) * p.H;
  if (blockIdx.y < 4) {
    float* const outs[4] = {p.dweight, p.dbias, p.dpost_weight, p.dpost_bias};
    float* dst = outs[blockIdx.y];
    if (!dst) return;
    detail::column_sum_cta(nullptr, p.ws + blockIdx.y * vec, p.teams, p.H, dst, p.H, blockIdx.x, smem);
    return;
  }
  const int c = static_cast<int>(blockIdx.y) - 3;
  const int64_t R = p.rows_per_team, at = c * R;      // first row of team c
  const int64_t gr = p.gate_rows ? p.gate_rows : p.rows;
  const int64_t g = at / gr, g0 = g * gr, g1 = min(int64_t(p.rows), g0 + gr);
  if (g0 >= at || g0 / R != c - 1) return;            // starts here, or crossed in earlier
  const int last = static_cast<int>((g1 - 1) / R);
  detail::column_sum_cta(p.ws + 5 * vec + int64_t(c - 1) * p.H, p.ws + 4 * vec + int64_t(c) * p.H,
                         last - c + 1, p.H, p.dgate + g * p.H, p.H, blockIdx.x, smem);
}

template <class TX, bool kLayer, bool kPost>
inline cudaError_t launch_block_norm(const NormParams& p, const Geometry& g, cudaStream_t s) {
  auto* kernel = g.cluster == 1 ? block_norm_kernel<TX, kLayer, kPost, 1>
                                : block_norm_kernel<TX, kLayer, kPost, 2>;
  return detail::launch_pdl(kernel, dim3(p.teams * g.cluster), dim3(g.threads), 0, s, p);
}

template <class TX, bool kLayer, bool kPost, bool kGate>
inline cudaError_t launch_block_norm_backward(const NormBackwardParams& p, const Geometry& g,
                                              cudaStream_t s) {
  auto* kernel = g.cluster == 1 ? block_norm_backward_kernel<TX, kLayer, kPost, kGate, 1>
                                : block_norm_backward_kernel<TX, kLayer, kPost, kGate, 2>;
  return detail::launch_pdl(kernel, dim3(p.teams * g.cluster), dim3(g.threads), 0, s, p);
}

}  // namespace norm_detail

inline cudaError_t block_norm(const blackhole_sm100_block_norm_args& a, cudaStream_t stream) {
  using namespace norm_detail;
  cudaError_t e = block_norm_check(a);
  if (e != cudaSuccess) return e;
  const Geometry g = geometry(a.H);
  NormParams p;
  p.x = a.x; p.o = a.o; p.gate = a.gate; p.weight = a.weight; p.bias = a.bias;
  p.post_weight = a.post_weight; p.post_bias = a.post_bias;
  p.h = a.h; p.out = a.out; p.sf = static_cast<uint8_t*>(a.sf); p.stats = a.stats;
  p.rows = a.rows; p.H = a.H; p.slice = g.slice;
  p.teams = std::min(a.rows, 148 * 16);
  p.gate_rows = a.gate ? a.gate_rows : 0;
  p.param_bf16 = a.param_is_bf16; p.gate_bf16 = a.gate_is_bf16; p.out_format = a.out_format;
  p.scale = a.scale; p.eps = a.eps; p.global_scale = a.global_scale;
  const bool layer = a.kind == 1, post = a.post_norm != 0;
  if (a.x_is_bf16) {
    using T = __nv_bfloat16;
    e = layer ? (post ? launch_block_norm<T, true, true>(p, g, stream) : launch_block_norm<T, true, false>(p, g, stream))
              : (post ? launch_block_norm<T, false, true>(p, g, stream) : launch_block_norm<T, false, false>(p, g, stream));
  } else {
    using T = float;
    e = layer ? (post ? launch_block_norm<T, true, true>(p, g, stream) : launch_block_norm<T, true, false>(p, g, stream))
              : (post ? launch_block_norm<T, false, true>(p, g, stream) : launch_block_norm<T, false, false>(p, g, stream));
  }
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}

inline cudaError_t block_norm_backward(const blackhole_sm100_block_norm_backward_args& a,
                                       cudaStream_t stream) {
  using namespace norm_detail;
  cudaError_t e = block_norm_backward_check(a);
  if (e != cudaSuccess) return e;
  const Geometry g = geometry(a.H);
  const Teams t = backward_teams(a.rows, a.H);
  NormBackwardParams p;
  p.h = a.h; p.dy = a.dy; p.dh = a.dh; p.o = a.o; p.gate = a.gate; p.weight = a.weight;
  p.post_weight = a.post_weight; p.post_bias = a.post_bias; p.stats = a.stats;
  p.dx = a.dx; p.d_o = a.d_o;
  p.dweight = a.dweight; p.dbias = a.dbias; p.dpost_weight = a.dpost_weight;
  p.dpost_bias = a.dpost_bias; p.dgate = a.dgate;
  p.ws = static_cast<float*>(a.workspace);
  p.rows = a.rows; p.H = a.H; p.slice = g.slice; p.teams = t.teams; p.rows_per_team = t.rows_per_team;
  p.gate_rows = a.gate ? a.gate_rows : 0;
  p.param_bf16 = a.param_is_bf16; p.gate_bf16 = a.gate_is_bf16;
  p.scale = a.scale;
  auto run = [&](auto tx) {
    using T = decltype(tx);
    const int sel = (a.kind == 1 ? 4 : 0) + (a.post_norm ? 2 : 0) + (a.gate ? 1 : 0);
    switch (sel) {
      case 0: return launch_block_norm_backward<T, false, false, false>(p, g, stream);
      case 1: return launch_block_norm_backward<T, false, false, true>(p, g, stream);
      case 2: return launch_block_norm_backward<T, false, true, false>(p, g, stream);
      case 3: return launch_block_norm_backward<T, false, true, true>(p, g, stream);
      case 4: return launch_block_norm_backward<T, true, false, false>(p, g, stream);
      case 5: return launch_block_norm_backward<T, true, false, true>(p, g, stream);
      case 6: return launch_block_norm_backward<T, true, true, false>(p, g, stream);
      default: return launch_block_norm_backward<T, true, true, true>(p, g, stream);
    }
  };
  e = a.x_is_bf16 ? run(__nv_bfloat16{}) : run(float{});
  if (e != cudaSuccess) return e;
  const bool edges = a.dgate && p.gate_rows != 1 && t.teams > 1;
  if (a.dweight || a.dbias || a.dpost_weight || a.dpost_bias || edges) {
    const dim3 grid((a.H + 31) / 32, 4 + (edges ? t.teams - 1 : 0));
    e = detail::launch_pdl(block_norm_sums_kernel, grid, dim3(1024), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

#endif  // __CUDACC__

}  // namespace blackhole::sm100
